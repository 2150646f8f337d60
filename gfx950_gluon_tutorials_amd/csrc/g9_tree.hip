// Attention of drafted tokens over a paged cache (g9_tree_fwd,
// include/gfx950_fmha.h); one node per request is plain decoding.
//
// Bound by reading the cache: every K and V row of the batch once, a few
// products per value.  So the kernel is a stream.  The work is a line of tiles:
// for each request, K/V head and block of 32 query rows (all query heads of
// the K/V head and all nodes, node-major) the tiles of 4096 / D keys from first
// to last.  The line is cut into equal parts, one per wave of a grid that fills
// the chip once: requests of any lengths load every CU alike, and a single long
// request is spread over all of them.  A wave keeps its own tiles in LDS (two
// stages of 8 KB of K and 8 KB of V, filled by LDS-DMA), so no wave ever waits
// for another one: there is no barrier in the loop.
//
// Blocks of 32 rows are half empty where a request brings fewer, which costs
// nothing: the matrix unit is idle most of the time (g9_wave.hpp has the tile).
//
// A block of rows whose tiles lie in one wave's part is finished there.  Else
// each wave writes its unnormalized sum, maximum and weight to the workspace and
// g9_tree_join, launched behind, joins them in the order of the keys: the result
// depends on no timing.
#include "../../include/gfx950_fmha.h"
#include "g9_attn_host.hpp"
#include "g9_wave.hpp"

namespace g9 {
namespace tree {

using namespace fa;

constexpr int kWgs = 256;  // one workgroup per CU

struct Params {
  const char* q;
  const char* kc;
  const char* vc;
  char* o;
  float* lse;                                      // [HQ][T], or null
  const int* table;
  const int* lengths;
  const int* cu;
  const unsigned long long* mask;                  // or null: a chain
  float* part;                                     // sums [2 kWorkers][kBlock][D], then (m, l) pairs
  struct Start* start;                             // [kWorkers]: where each part begins
  long long q_t, q_h, o_t, o_h;                    // token / head strides, bytes
  long long k_b, k_h, v_b, v_h;                    // block / head strides, bytes
  long long table_stride;
  u32 k_t, v_t;                                    // token strides, bytes
  int num_blocks, width, shift, words;
  int B, T, HQ, HK, group;
  float scale_log2;

  // A query row: its node (-1: no row), its request's context and first query.
  struct Row {
    int node, context, q0;
  };
  // Bit i: the row reads key k0 + i of `keys`.
  G9_DEV unsigned long long reads(const Row& r, int k0, int keys) const {
    const int n0 = max(k0 - r.context, -4096);  // key k0's node, negative in the context
    unsigned long long w;
    if (!mask) {
      const int c = r.node + 1 - n0;  // keys up to the row's own
      w = c >= 64 ? ~0ull : c <= 0 ? 0 : (1ull << c) - 1;
    } else {
      const int first = max(n0, 0) >> 6, sh = max(n0, 0) & 63;
      const unsigned long long* const m = mask + (long long)(r.q0 + max(r.node, 0)) * words + first;
      const unsigned long long a = first < words ? m[0] : 0, b = first + 1 < words ? m[1] : 0;
      w = sh ? a >> sh | b << (64 - sh) : a;
      if (n0 < 0) w = n0 <= -64 ? ~0ull : w << -n0 | ((1ull << -n0) - 1);
    }
    const int left = keys - k0;
    if (left < 64) w &= left <= 0 ? 0 : (1ull << left) - 1;
    return w;
  }
};

// One request: its query rows, context, keys, blocks of query rows, tiles.
struct Req {
  int q0, n, context, keys, blocks, tiles;
};
// A place on the line.
struct Place {
  Req r;
  int b, hk, block, tile;
};
// The beginning of a worker's part, for the kernel that joins the parts.
struct alignas(32) Start {
  int q0, n, hk, block, tile, tiles;
  u32 total_lo, total_hi;
};

// x / y with the 32-bit division where it holds them.
G9_DEV unsigned long long quotient(unsigned long long x, unsigned long long y) {
  return (x | y) >> 32 ? x / y : (unsigned long long)((u32)x / (u32)y);
}

G9_DEV void make_uniform(Place& a) {
  for (int* x : {&a.r.q0, &a.r.n, &a.r.context, &a.r.keys, &a.r.blocks, &a.r.tiles, &a.b, &a.hk, &a.block, &a.tile})
    *x = uniform(*x);
}

// The line of tiles: KEYS keys a tile, blocks of BLOCK query rows, WORKERS parts.
// A block's tiles have LEAD places without work before them, for what its
// beginning and end cost: else the parts of many short requests take longest.
template <int KEYS, int BLOCK, int WORKERS, int LEAD>
struct Line {
  static constexpr int kKeys = KEYS, kBlock = BLOCK, kWorkers = WORKERS, kLead = LEAD;

  static G9_DEV Req request(const Params& p, int b) {
    Req r;
    r.q0 = min(max(p.cu[b], 0), p.T);
    r.n = min(max(p.cu[b + 1], r.q0), p.T) - r.q0;
    r.context = max(p.lengths[b], 0);
    r.keys = (int)min((long long)r.context + r.n, (long long)p.width << p.shift);
    r.blocks = (int)(((long long)r.n * p.group + kBlock - 1) / kBlock);
    r.tiles = max((r.keys + kKeys - 1) / kKeys, 1);
    return r;
  }
  static G9_DEV unsigned long long tiles_of(const Params& p, const Req& r) {
    return (unsigned long long)r.blocks * (unsigned)p.HK * (unsigned)(kLead + r.tiles);
  }
  // Worker w of W takes the places [w n / W, (w + 1) n / W) of a line of n; W is at
  // most n, so that no part in between is empty.
  static G9_DEV unsigned workers(unsigned long long n) { return n < kWorkers ? (unsigned)n : kWorkers; }
  static G9_DEV unsigned long long part_begin(unsigned w, unsigned long long n) { return quotient(w * n, workers(n)); }
  static G9_DEV unsigned worker_of(unsigned long long place, unsigned long long n) {
    return (unsigned)quotient((place + 1) * workers(n) - 1, n);
  }

  // This worker's first tile, and the places of its part from there on (none or
  // less: no tile).  The workgroup sums the requests' places into LDS (first[B + 1]).
  template <int THREADS>
  static G9_DEV int locate(const Params& p, char* smem, unsigned worker, Place& at) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    unsigned long long* const first = reinterpret_cast<unsigned long long*>(smem);  // then the waves' sums
    unsigned long long* const sums = first + p.B + 1;
    const int run = (p.B + THREADS - 1) / THREADS;
    const int b0 = min(tid * run, p.B), b1 = min(b0 + run, p.B);
    unsigned long long mine = 0;
    for (int b = b0; b < b1; ++b) mine += tiles_of(p, request(p, b));
    unsigned long long before = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const unsigned long long x = __shfl_up(before, d, 64);
      if (lane >= d) before += x;
    }
    if (lane == 63) sums[wave] = before;
    __syncthreads();
    before -= mine;
    unsigned long long total = 0;
    for (int w = 0; w < THREADS / 64; ++w) {
      if (w < wave) before += sums[w];
      total += sums[w];
    }
    for (int b = b0; b < b1; ++b) {
      first[b] = before;
      before += tiles_of(p, request(p, b));
    }
    if (tid == 0) first[p.B] = total;
    __syncthreads();
    total = uniform(total);
    int left = 0;
    if (worker < workers(total)) {
      const unsigned long long begin = uniform(part_begin(worker, total));
      left = uniform((int)(part_begin(worker + 1, total) - begin));
      // The last request that begins at or before the part (empty ones begin
      // where the next one does).
      int lo = 0, hi = p.B;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (first[mid] <= begin)
          lo = mid;
        else
          hi = mid;
      }
      at.b = uniform(lo);
      at.r = request(p, at.b);
      const unsigned long long in = uniform(begin - first[lo]);
      const unsigned long long unit = quotient(in, (unsigned)(kLead + at.r.tiles));
      const int place = (int)(in - unit * (unsigned)(kLead + at.r.tiles));
      at.tile = max(place - kLead, 0);
      left -= uniform(max(kLead - place, 0));
      at.hk = (int)quotient(unit, (unsigned)at.r.blocks);
      at.block = (int)(unit - (unsigned long long)at.hk * at.r.blocks);
      make_uniform(at);
    }
    // Worker 0 says how long the line is, also where it is empty.
    if ((worker == 0 || worker < workers(total)) && (THREADS == 64 * (kWorkers / kWgs) ? lane == 0 : tid == 0))
      p.start[worker] = {at.r.q0, at.r.n, at.hk, at.block, at.tile, at.r.tiles, (u32)total, (u32)(total >> 32)};
    __syncthreads();  // first[] is read: what comes next takes its place
    return left;
  }
  // The first tile of the block behind `a`'s (there is one).
  static G9_DEV Place next_block(const Params& p, const Place& a) {
    Place n = a;
    n.tile = 0;
    if (++n.block < n.r.blocks) return n;
    n.block = 0;
    if (++n.hk < p.HK) return n;
    n.hk = 0;
    do {
      n.b = min(n.b + 1, p.B - 1);
      n.r = request(p, n.b);
    } while (n.r.blocks == 0 && n.b < p.B - 1);
    make_uniform(n);
    return n;
  }
  // To the part's next tile, if it has one.
  static G9_DEV bool advance(const Params& p, Place& a, int& left) {
    const bool end = a.tile + 1 == a.r.tiles;
    left -= end ? 1 + kLead : 1;
    if (left <= 0) return false;
    if (end)
      a = next_block(p, a);
    else
      ++a.tile;
    return true;
  }
};
// A wave's own tiles of up to 8 KB, or a workgroup's of 16 KB.  A block costs a
// wave nothing beside its tiles that shows (1 to 3 places: 0 to 5% slower); a
// workgroup it costs as much as 384 keys (us, blocks of 256 rows of head dim 128,
// 64 rows a request, with and without the places: 64 x 100-8192 tokens 243 and
// 331, 64 x 100-2000 96 and 140, 4 x 8000 with 200 x 100 96 and 148).
template <int HD, int NQ>
using Narrow = Line<4096 / HD, 32 * NQ, 4 * kWgs, 0>;
template <int HD>
using Wide = Line<8192 / HD, 256, kWgs, 384 * HD / 8192>;

// A lane's query row of the block.
template <class L>
G9_DEV Params::Row row_of(const Params& p, const Place& at, int row) {
  const int nd = (at.block * L::kBlock + row) / p.group;
  const bool in = nd < at.r.n;
  return {in ? nd : -1, at.r.context, at.r.q0};
}
template <class L>
G9_DEV const char* query_of(const Params& p, const Place& at, int row, int node) {
  const int hd = at.block * L::kBlock + row - max(node, 0) * p.group;
  return p.q + (long long)(at.r.q0 + max(node, 0)) * p.q_t + (long long)(at.hk * p.group + (node < 0 ? 0 : hd)) * p.q_h;
}
// The row's results, or its sum to slot `slot` of the workspace.  o, m, l as the
// 32x32 layout leaves them: lane half h has the values 8 r + 4 h + 0..3 of every
// 32, l is its half of the weight.
template <bool BF16, int HD, class L>
G9_DEV void finish(const Params& p, const Place& at, int slot, int row, int node, const f32x16 (&o)[HD / 32], float m,
                   float l) {
  const int h = (threadIdx.x & 63) >> 5;
  const float lt = xhalf(l, [](float x, float y) { return x + y; });
  if (node < 0) return;
  if (slot >= 0) {
    float* const sum = p.part + ((size_t)slot * L::kBlock + row) * HD;
#pragma unroll
    for (int d = 0; d < HD / 32; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        *reinterpret_cast<f32x4*>(sum + 32 * d + 8 * r + 4 * h) =
            f32x4{o[d][4 * r], o[d][4 * r + 1], o[d][4 * r + 2], o[d][4 * r + 3]};
    if (h == 0) {
      float* const ml = p.part + (size_t)2 * L::kWorkers * L::kBlock * HD + ((size_t)slot * L::kBlock + row) * 2;
      ml[0] = m, ml[1] = lt;
    }
    return;
  }
  const int hq = at.hk * p.group + at.block * L::kBlock + row - node * p.group;
  const long long tok = at.r.q0 + node;
  // By its bits: comparisons here may take NaN for a number.
  const bool none = (__float_as_uint(lt) << 1) == 0;
  const float inv = none ? 0.f : 1.f / lt;
  char* const orow = p.o + tok * p.o_t + hq * p.o_h;
#pragma unroll
  for (int d = 0; d < HD / 32; ++d)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      *reinterpret_cast<u32x2*>(orow + (32 * d + 8 * r + 4 * h) * 2) =
          u32x2{pack2<BF16>(o[d][4 * r] * inv, o[d][4 * r + 1] * inv),
                pack2<BF16>(o[d][4 * r + 2] * inv, o[d][4 * r + 3] * inv)};
  if (p.lse && h == 0) p.lse[(long long)hq * p.T + tok] = none ? -__builtin_inff() : (m + __builtin_log2f(lt)) * kLn2;
}

// Consecutive workgroups go round the 8 XCDs; consecutive parts of the line stay
// on one, whose L2 then serves the blocks of rows that share keys.
G9_DEV unsigned my_part() { return (blockIdx.x & 7) * (kWgs / 8) + (blockIdx.x >> 3); }

// The 16-row pieces' pages of a tile; -1: none.
template <class W>
G9_DEV void pages_of(const Params& p, const Place& at, int (&pg)[W::kPieces]) {
#pragma unroll
  for (int i = 0; i < W::kPieces; ++i) {
    const int k = at.tile * W::kKeys + 16 * i;
    pg[i] = k < at.r.keys ? p.table[at.b * p.table_stride + (k >> p.shift)] : -1;
  }
}
template <class W>
G9_DEV void fill(const Params& p, const W& w, const Place& at, const int (&pg)[W::kPieces], int stage) {
#pragma unroll
  for (int i = 0; i < W::kPieces; ++i) {
    const int k = at.tile * W::kKeys + 16 * i, off = k & ((1 << p.shift) - 1);
    const bool in = (u32)pg[i] < (u32)p.num_blocks;
    const int rows = in ? min(max(at.r.keys - k, 0), 16) : 0;
    const long long page = in ? pg[i] : 0;
    w.fill_piece(i, stage, p.kc + page * p.k_b + at.hk * p.k_h + (unsigned long long)off * p.k_t,
                 p.vc + page * p.v_b + at.hk * p.v_h + (unsigned long long)off * p.v_t, rows, p.k_t, p.v_t);
  }
}
template <class W, class L, int NQ>
G9_DEV void begin(const Params& p, W& w, const Place& at) {
#pragma unroll
  for (int t = 0; t < NQ; ++t) {
    w.node[t] = row_of<L>(p, at, 32 * t + w.col).node;
    w.load_q(t, query_of<L>(p, at, 32 * t + w.col, w.node[t]));
  }
  w.clear();
  w.context = at.r.context, w.q0 = at.r.q0, w.keys = at.r.keys;
  // Waited for here: the compiler does not count the DMAs in flight, and a wait
  // of its own at the first use would be one in every tile.
  waitcnt<0, 0>();
}

template <bool BF16, int HD, int NQ>
G9_DEV void narrow(const Params& p, char* smem) {
  using W = Wave<Params, BF16, HD, NQ>;
  using L = Narrow<HD, NQ>;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned worker = my_part() * 4 + wave;
  Place cur{};
  int left = L::template locate<256>(p, smem, worker, cur);
  if (left <= 0) return;

  W w(p);
  w.init(smem, wave, p.k_t, p.v_t);
  int pg[W::kPieces];
  pages_of<W>(p, cur, pg);
  fill(p, w, cur, pg, 0);
  Place nxt = cur;
  bool more = L::advance(p, nxt, left);  // nxt is a tile
  if (more) pages_of<W>(p, nxt, pg);
  bool fresh = true, from_start = cur.tile == 0;
  for (int i = 0;; ++i) {
    // The stage that tile i + 1 takes was last read for tile i - 1.
    waitcnt<63, 0>();
    __builtin_amdgcn_sched_barrier(0);
    Place aft = nxt;
    bool more_aft = false;
    if (more) {
      fill(p, w, nxt, pg, (i + 1) & 1);
      more_aft = L::advance(p, aft, left);
      if (more_aft) pages_of<W>(p, aft, pg);
      if (fresh) begin<W, L, NQ>(p, w, cur);
      waitcnt<2 * W::kDmas, 15>();
    } else {
      if (fresh) begin<W, L, NQ>(p, w, cur);
      waitcnt<0, 15>();
    }
    __builtin_amdgcn_sched_barrier(0);
    const bool tail = (cur.tile + 1) * W::kKeys > min(cur.r.context, cur.r.keys);
    w.tile(cur.tile * W::kKeys, i & 1, tail);
    const bool last = cur.tile + 1 == cur.r.tiles;
    fresh = last;
    if (last || !more) {
      // Slot 0 of the worker: a block that another worker began; slot 1: one
      // that the next worker goes on with.
#pragma unroll
      for (int t = 0; t < NQ; ++t)
        finish<BF16, HD, L>(p, cur, last && from_start ? -1 : (int)(2 * worker + (from_start ? 1 : 0)), 32 * t + w.col,
                            w.node[t], w.o[t], w.m[t], w.l[t]);
      from_start = true;
    }
    if (!more) break;
    cur = nxt;
    nxt = aft;
    more = more_aft;
  }
}

// Many query rows: a workgroup's 8 waves, 32 rows each, share every tile, on the
// pipeline of g9_fmha_pipe.hpp.
template <bool BF16, int HD>
struct WidePipe {
  using T = Pipe<Params, BF16, true, false, HD, kPaged>;
  static constexpr int kLds = T::kLdsBytes + kWaves * T::kScratchBytes;
};

// The kernel's argument, read again (scalar loads) where the compiler cannot take
// it for what it has: what only a block's beginning and end need is not held, and
// spilled, through the loop.
G9_DEV Params again() {
  typedef const u32 __attribute__((address_space(4))) Const;
  struct Words {
    u32 w[sizeof(Params) / 4];
  } x;
  Const* a = (Const*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(a));
#pragma unroll
  for (unsigned i = 0; i < sizeof(Params) / 4; ++i) x.w[i] = a[i];
  Params p = __builtin_bit_cast(Params, x);
  const auto global = [](auto*& t) {
    typedef std::remove_reference_t<decltype(*t)> T;
    t = (T*)(__attribute__((address_space(1))) T*)t;
  };
  global(p.q), global(p.kc), global(p.vc), global(p.o), global(p.lse), global(p.table), global(p.part);
  return p;
}

template <bool BF16, int HD>
G9_DEV void wide(const Params& p, char* smem) {
  using L = Wide<HD>;
  using PipeT = typename WidePipe<BF16, HD>::T;
  static_assert(PipeT::kBN == L::kKeys && kBlockM == L::kBlock);
  const unsigned worker = my_part();
  Place cur{};
  int left = L::template locate<kThreads>(p, smem, worker, cur);
  const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5;
  PipeT P(p);
  P.wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  P.lds0 = (u32)(uintptr_t)to_lds(smem);
  P.pscratch = smem + PipeT::kLdsBytes + P.wave * PipeT::kScratchBytes;
  P.sc = p.scale_log2;
  P.voffk = P.voff_k_of(lane), P.voffv = P.voff_v_of(lane);
  P.ak = P.ak_of(lane), P.av = P.av_of(lane);
  const bool lag = P.wave >= 4;
  const int row = P.wave * 32 + (lane & 31);
  while (left > 0) {
    const int seg = min(left, cur.r.tiles - cur.tile);
    const Params pb = again();
    P.keys = min(cur.r.keys, (cur.tile + seg) * PipeT::kBN);
    P.wlim = min(cur.r.context, P.keys);
    P.t0 = cur.tile;
    P.table = pb.table + cur.b * pb.table_stride;
    P.row = row_of<L>(pb, cur, row);
    P.nte = max((seg + 1) & ~1, 2);
    P.kp = pb.kc + cur.hk * pb.k_h;
    P.vp = pb.vc + cur.hk * pb.v_h;
    const int nte = P.nte;
    const char* const qrow = query_of<L>(pb, cur, row, P.row.node);
#pragma unroll
    for (int s = 0; s < PipeT::kNS; ++s) P.qf[s] = *reinterpret_cast<const u32x4*>(qrow + (16 * s + 8 * h) * 2);
    // The prologue of g9_fmha.hip's kernel, with more tiles asked for.
    P.hold_pages(0);
    int pg[6];
#pragma unroll
    for (int i = 0; i < 6; ++i) pg[i] = P.page_of(i);
    const auto ask_k = [&](int tile, int page) {
      P.pgk = page;
      P.dma_k(tile, tile & 3);
    };
    const auto ask_v = [&](int tile, int page) {
      P.pgv = page;
      P.dma_v(tile, tile & 3);
    };
    ask_k(0, pg[0]);
    ask_v(0, pg[0]);
    ask_k(1, pg[1]);
#pragma unroll
    for (int d = 0; d < PipeT::kND; ++d) P.o[d] = f32x16{};
    P.m = -3.0e38f;
    P.l = 0.f;
    waitcnt<0, 0>();
    barrier();
    if (nte > 2) ask_k(2, pg[2]);
    ask_v(1, pg[1]);
    if (nte > 2) {
      ask_k(3, pg[3]);
      ask_v(2, pg[2]);
    }
    P.template read_k<-1>(0);
    typename PipeT::Sc sa, sb;
    P.qk(sa);
    waitcnt<63, 0>();
    barrier();  // every wave has read K_0: its buffer takes K_4
    if (nte > 4) ask_k(4, pg[4]);
    if (nte > 2) ask_v(3, pg[3]);
    P.pgv = pg[4];
    P.pgk = pg[5];
    if (P.masked(0)) P.mask_tile(sa, 0);
    P.vec0(sa);
    P.vec1(sa);
    P.l *= P.alpha;
    P.template read_k<-1>(1);
    waitcnt<63, 0>();
    if (lag) barrier();
    // A wave without query rows leaves the tiles to the others.
    const int own = (cur.block * L::kBlock + P.wave * 32) / pb.group < cur.r.n ? nte : 2;
    int j = 0;
    for (; j + 2 < own; j += 2) {
      P.template step<0, true>(j, sa, sb);
      P.template step<1, true>(j + 1, sb, sa);
    }
    P.template step<0, true>(j, sa, sb);
    P.template step<1, false>(j + 1, sb, sa);
    __builtin_amdgcn_s_setprio(0);
    for (j += 2; j < nte; ++j) P.idle(j);
    if (!lag) barrier();
    const bool from_start = cur.tile == 0, last = cur.tile + seg == cur.r.tiles;
    const Params pe = again();
    finish<BF16, HD, L>(pe, cur, last && from_start ? -1 : (int)(2 * worker + (from_start ? 1 : 0)), row, P.row.node, P.o,
                        P.m, P.l);
    left -= seg + L::kLead;
    if (left > 0) cur = L::next_block(pe, cur);
    barrier();  // the stages are read: the next block's tiles take them
  }
}

// The joined row: with m the largest of the parts' maxima, the sum of 2^(m_i - m)
// O_i over the sum of 2^(m_i - m) l_i, in the order of the keys.
template <bool BF16>
G9_DEV void store4(const Params& p, long long tok, int hq, int c, f32x4 sum, float m, float l) {
  const bool none = (__float_as_uint(l) << 1) == 0;
  const float inv = none ? 0.f : 1.f / l;
  *reinterpret_cast<u32x2*>(p.o + tok * p.o_t + hq * p.o_h + c * 8) =
      u32x2{pack2<BF16>(sum[0] * inv, sum[1] * inv), pack2<BF16>(sum[2] * inv, sum[3] * inv)};
  if (p.lse && c == 0) p.lse[(long long)hq * p.T + tok] = none ? -__builtin_inff() : (m + __builtin_log2f(l)) * kLn2;
}

// Joins the blocks that are cut.  A block of n parts has the n - 1 workers whose
// parts begin within it, and with each of them a workgroup here (blockIdx.x + 1):
// they (and gridDim.y times as many) share its rows, so that a workgroup's work
// is a fraction of a part, however many parts a long request's blocks have.
template <int HD>
constexpr int kJoinThreads = 4 * HD;
template <bool BF16, int HD, class L>
G9_DEV void join(const Params& p, float* lds) {
  const unsigned w = blockIdx.x + 1;
  const Start zero = p.start[0];
  const unsigned long long total = (unsigned long long)zero.total_hi << 32 | zero.total_lo;
  const Start st = p.start[w];  // asked for together with worker 0's
  if (w >= L::workers(total) || st.tile == 0) return;
  const unsigned long long u0 = L::part_begin(w, total) - (unsigned)st.tile;
  const unsigned w0 = L::worker_of(u0, total), n = L::worker_of(u0 + st.tiles - 1, total) - w0 + 1;
  // Worker w0, in whose part the block begins, has it in slot 1, the others in slot 0.
  const size_t head = (size_t)2 * w0 + 1;
  const float* const ml = p.part + (size_t)2 * L::kWorkers * L::kBlock * HD;
  const int row0 = st.block * L::kBlock;
  const u32 rows = (u32)min((long long)st.n * p.group - row0, (long long)L::kBlock);
  const u32 share = (w - w0 - 1) * gridDim.y + blockIdx.y, shares = (n - 1) * gridDim.y;
  const u32 from = share * rows / shares, to = (share + 1) * rows / shares;
  constexpr unsigned kCols = HD / 4, kLanes = kJoinThreads<HD> / kCols;
  const unsigned c = threadIdx.x % kCols, lane = threadIdx.x / kCols;
  f32x4 sum;
  float m, l;
  const auto clear = [&] { sum = f32x4{}, m = -3.0e38f, l = 0.f; };
  const auto add = [&](f32x4 x, float mk, float lk) {
    const float m_new = __builtin_fmaxf(m, mk);
    const float f = __builtin_amdgcn_exp2f(m - m_new), g = __builtin_amdgcn_exp2f(mk - m_new);
    l = l * f + lk * g;
    sum = sum * f + x * g;
    m = m_new;
  };
  // Adds the row's parts k0, k0 + step, ..., kAtOnce of them asked for together.
  const auto add_parts = [&]<unsigned kAtOnce>(unsigned in, unsigned k0, unsigned step) {
    for (unsigned k = k0; k < n; k += kAtOnce * step) {
      float mk[kAtOnce], lk[kAtOnce];
      f32x4 x[kAtOnce];
#pragma unroll
      for (unsigned e = 0; e < kAtOnce; ++e) {
        const unsigned i = min(k + e * step, n - 1);
        const size_t a = (i ? (size_t)2 * (w0 + i) : head) * L::kBlock + in;
        mk[e] = ml[a * 2], lk[e] = ml[a * 2 + 1];
        x[e] = *reinterpret_cast<const f32x4*>(p.part + a * HD + 4 * c);
      }
#pragma unroll
      for (unsigned e = 0; e < kAtOnce; ++e)
        if (k + e * step < n) add(x[e], mk[e], lk[e]);
    }
  };
  const auto store = [&](unsigned in) {
    const int row = row0 + (int)in, nd = row / p.group;
    store4<BF16>(p, st.q0 + nd, st.hk * p.group + row - nd * p.group, c, sum, m, l);
  };
  // Round trips to memory: a row per 16-byte column group of threads, its parts
  // eight at a time, or the threads sharing a row's parts, and the row's join in
  // LDS behind them.
  const u32 r = to - from;
  if ((r + kLanes - 1) / kLanes * ((n + 7) / 8) <= 2 * r) {
    for (unsigned in = from + lane; in < to; in += kLanes) {
      clear();
      if (n <= 3)
        add_parts.template operator()<3>(in, 0, 1);
      else
        add_parts.template operator()<8>(in, 0, 1);
      store(in);
    }
    return;
  }
  for (unsigned in = from; in < to; ++in) {
    clear();
    add_parts.template operator()<8>(in, lane, kLanes);
    float* const mine = lds + threadIdx.x * 7;
#pragma unroll
    for (int e = 0; e < 4; ++e) mine[e] = sum[e];
    mine[4] = m, mine[5] = l;
    __syncthreads();
    if (lane == 0) {
      for (unsigned i = 1; i < kLanes; ++i) {
        const float* const o = lds + (i * kCols + c) * 7;
        add(f32x4{o[0], o[1], o[2], o[3]}, o[4], o[5]);
      }
      store(in);
    }
    __syncthreads();
  }
}

}  // namespace tree
}  // namespace g9

using namespace g9;
using namespace g9::host;

// The bound of 512 threads (256 are launched) keeps the kernels to 256 registers a
// lane, all of the vector file: with more the products' results go to the
// accumulation file, and a third of a tile's instructions moves them back.
#define G9_TREE_NARROW(NAME, BF16, HD, NQ)                                                                    \
  extern "C" __global__ __launch_bounds__(512) void                                                           \
  g9_tree_##NAME(tree::Params p) {                                                                            \
    __shared__ __attribute__((aligned(1024))) char smem[4 * fa::Wave<tree::Params, BF16, HD, NQ>::kWaveLds];               \
    tree::narrow<BF16, HD, NQ>(p, smem);                                                                      \
  }                                                                                                           \
  extern "C" __global__ __launch_bounds__(tree::kJoinThreads<HD>) void g9_tree_join_##NAME(tree::Params p) {  \
    __shared__ float lds[tree::kJoinThreads<HD> * 7];                                                         \
    tree::join<BF16, HD, tree::Narrow<HD, NQ>>(p, lds);                                                       \
  }
#define G9_TREE_WIDE(NAME, BF16, HD)                                                                          \
  extern "C" __global__ __launch_bounds__(fa::kThreads) __attribute__((amdgpu_waves_per_eu(2, 2))) void       \
  g9_tree_##NAME(tree::Params p) {                                                                            \
    __shared__ __attribute__((aligned(1024))) char smem[tree::WidePipe<BF16, HD>::kLds];                       \
    tree::wide<BF16, HD>(p, smem);                                                                            \
  }                                                                                                           \
  extern "C" __global__ __launch_bounds__(tree::kJoinThreads<HD>) void g9_tree_join_##NAME(tree::Params p) {  \
    __shared__ float lds[tree::kJoinThreads<HD> * 7];                                                         \
    tree::join<BF16, HD, tree::Wide<HD>>(p, lds);                                                             \
  }
G9_TREE_NARROW(bf16_q32, true, 128, 1)
G9_TREE_NARROW(f16_q32, false, 128, 1)
G9_TREE_NARROW(bf16_d64_q32, true, 64, 1)
G9_TREE_NARROW(f16_d64_q32, false, 64, 1)
G9_TREE_NARROW(bf16_d64_q64, true, 64, 2)
G9_TREE_NARROW(f16_d64_q64, false, 64, 2)
G9_TREE_WIDE(bf16_q256, true, 128)
G9_TREE_WIDE(f16_q256, false, 128)
G9_TREE_WIDE(bf16_d64_q256, true, 64)
G9_TREE_WIDE(f16_d64_q256, false, 64)

namespace {

// Query rows of a block, by the rows that the requests of a batch bring on
// average to one K/V head.  Measured (us a call, blocks of 32, 64 and 256 rows;
// 8 K/V heads, a cache that no last level holds, one MI355X):
//   head dim 64     16 x 6000 tokens    64 x 100-8192     256 x 200-600
//     32 rows        62   69   62       149  166  173      73   80  136
//     64 rows        99   72   66       262  175  177     116   88  141
//     96 rows       133  117   70       375  301  183     160  143  155
//     128 rows      147  118   73       497  304  196     206  152  162
//   head dim 128 (blocks of 64 do not fit its registers)
//     32 rows       100    -   96       248    -  230     125    -  139
//     64 rows       155    -   97       460    -  240     204    -  151
//     128 rows      239    -  105       876    -  268     361    -  179
// and 1 x 700 tokens, 32 rows: 15 and 21 (head dim 64), 19 and 22.
enum { Q32, Q64, Q256 };
int form_of(int64_t B, int64_t T, int64_t group, int64_t D) {
  const int64_t rows = (T + B - 1) / B * group;
  return rows <= 32 ? Q32 : D == 64 && rows <= 64 ? Q64 : Q256;
}
// The sums of 2 x 1024 blocks of 32 or 64 rows, or of 2 x 256 of 256.
size_t part_floats(int form, int64_t D) { return (size_t)2 * (form == Q32 ? 1024 * 32 : 1024 * 64) * (D + 2); }

#define G9_TREE_FN(WHAT, Q) {reinterpret_cast<const void*>(WHAT##f16_##Q), reinterpret_cast<const void*>(WHAT##bf16_##Q)}
#define G9_TREE_FN64(WHAT, Q) \
  {reinterpret_cast<const void*>(WHAT##f16_d64_##Q), reinterpret_cast<const void*>(WHAT##bf16_d64_##Q)}
// [form][head dim 64][bf16]
const void* const kRun[3][2][2] = {{G9_TREE_FN(g9_tree_, q32), G9_TREE_FN64(g9_tree_, q32)},
                                   {{nullptr, nullptr}, G9_TREE_FN64(g9_tree_, q64)},
                                   {G9_TREE_FN(g9_tree_, q256), G9_TREE_FN64(g9_tree_, q256)}};
const void* const kJoin[3][2][2] = {{G9_TREE_FN(g9_tree_join_, q32), G9_TREE_FN64(g9_tree_join_, q32)},
                                    {{nullptr, nullptr}, G9_TREE_FN64(g9_tree_join_, q64)},
                                    {G9_TREE_FN(g9_tree_join_, q256), G9_TREE_FN64(g9_tree_join_, q256)}};

// The workspace: sums, then start[].
size_t start_at(int form, int64_t D) { return (part_floats(form, D) * 4 + 31) / 32 * 32; }
size_t workspace_of(int form, int64_t D) { return start_at(form, D) + 1024 * sizeof(tree::Start); }

}  // namespace

extern "C" size_t g9_tree_workspace_size(int64_t B, int64_t T, int64_t HQ, int64_t HK, int64_t D) {
  if (B <= 0 || T <= 0 || HQ <= 0 || HK <= 0 || HQ % HK || D <= 0) return 0;
  return workspace_of(form_of(B, T, HQ / HK, D), D);
}

extern "C" int g9_tree_fwd(const void* q, const void* k_cache, const void* v_cache, void* o, float* lse,
                const int32_t* block_table, int64_t table_stride, int64_t width, const int32_t* lengths,
                const int32_t* cu_q, const int64_t* tree_mask, int64_t words, int64_t B, int64_t T, int64_t HQ,
                int64_t HK, int64_t D, int64_t num_blocks, int64_t block_size, const int64_t* q_strides,
                const int64_t* kc_strides, const int64_t* vc_strides, const int64_t* o_strides, float sm_scale,
                int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  if (dtype != G9_F16 && dtype != G9_BF16) return G9_ERR_DTYPE;
  if (B < 0 || B > G9_TREE_MAX_REQUESTS || T < 0 || T > kMaxRows || HQ <= 0 || HQ > 65536 || HK <= 0 || HQ % HK ||
      (D != 64 && D != 128) || !scale_ok(sm_scale) || num_blocks < 0 || num_blocks > kMaxRows || width < 0 ||
      width > kMaxRows || !block_size_ok(block_size) || width * block_size > (int64_t(1) << 30) || words < 0 || words > 1024 ||
      (tree_mask && words == 0))
    return G9_ERR_SHAPE;
  if (!q_strides || !kc_strides || !vc_strides || !o_strides) return G9_ERR_LAYOUT;
  if (!steps(q_strides, 2) || !steps(kc_strides, 3) || !steps(vc_strides, 3) || !steps(o_strides, 2))
    return G9_ERR_LAYOUT;
  const int64_t size[2] = {T, HQ};
  if (!apart(size, o_strides, 2, D) || (B > 1 && table_stride < width)) return G9_ERR_LAYOUT;
  // A 16-row piece of a page lies within a descriptor's range, its rows apart.
  for (const int64_t* st : {kc_strides, vc_strides})
    if (st[1] < D || st[1] * 2 * 16 >= (int64_t(1) << 31)) return G9_ERR_LAYOUT;
  if (T * HQ > INT32_MAX) return G9_ERR_SHAPE;
  if (B == 0 || T == 0) return G9_OK;
  if (!q || !o || !lengths || !cu_q || (width && !block_table) || (num_blocks && (!k_cache || !v_cache)))
    return G9_ERR_LAYOUT;
  if (!aligned16(q) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(o) || ((uintptr_t)lse & 3) ||
      ((uintptr_t)tree_mask & 7))
    return G9_ERR_LAYOUT;
  const int64_t group = HQ / HK;
  const int form = form_of(B, T, group, D);
  if (!workspace || ((uintptr_t)workspace & 31) || workspace_bytes < workspace_of(form, D)) return G9_ERR_WORKSPACE;
  tree::Params p{};
  p.q = static_cast<const char*>(q);
  p.kc = static_cast<const char*>(k_cache);
  p.vc = static_cast<const char*>(v_cache);
  p.o = static_cast<char*>(o);
  p.lse = lse;
  p.table = block_table;
  p.lengths = lengths;
  p.cu = cu_q;
  p.mask = reinterpret_cast<const unsigned long long*>(tree_mask);
  p.part = static_cast<float*>(workspace);
  p.start = reinterpret_cast<tree::Start*>(static_cast<char*>(workspace) + start_at(form, D));
  p.q_t = q_strides[0] * 2, p.q_h = q_strides[1] * 2, p.o_t = o_strides[0] * 2, p.o_h = o_strides[1] * 2;
  p.k_b = kc_strides[0] * 2, p.k_h = kc_strides[2] * 2, p.v_b = vc_strides[0] * 2, p.v_h = vc_strides[2] * 2;
  p.k_t = (u32)(kc_strides[1] * 2), p.v_t = (u32)(vc_strides[1] * 2);
  p.table_stride = table_stride;
  p.num_blocks = (int)num_blocks, p.width = (int)width, p.shift = log2_of(block_size), p.words = (int)words;
  p.B = (int)B, p.T = (int)T, p.HQ = (int)HQ, p.HK = (int)HK, p.group = (int)group;
  p.scale_log2 = sm_scale * fa::kLog2e;
  void* args[] = {&p};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const int d64 = D == 64, bf16 = dtype == G9_BF16;
  if (hipLaunchKernel(kRun[form][d64][bf16], dim3(tree::kWgs), dim3(form == Q256 ? fa::kThreads : 256), args, 0, st) !=
      hipSuccess)
    return G9_ERR_HIP;
  return launched(hipLaunchKernel(kJoin[form][d64][bf16], dim3(form == Q256 ? 255 : 1023, form == Q256 ? 4 : 1),
                                  dim3(unsigned(4 * D)), args, 0, st));
}
