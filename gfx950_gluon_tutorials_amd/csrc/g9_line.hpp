// The work of the attentions over a paged cache (g9_tree.hip, g9_latent.hip) as a
// line of key tiles, cut into equal parts: which tiles a worker takes follows from
// the requests' lengths alone, and every worker finds its part itself.  Which keys a
// query row reads; and how the parts of a row come together.
#pragma once

#include "g9_wave.hpp"

namespace g9 {
namespace fa {

constexpr int kWgs = 256;  // one workgroup per CU

// A query row: its node (-1: no row), its request's context and first query.
struct NodeRow {
  int node, context, q0;
};
// Bit i: the row reads key k0 + i of `keys`, the context's and those of the nodes
// that p.mask names (p.words words a node; none: a chain).
template <class Params>
G9_DEV unsigned long long node_reads(const Params& p, const NodeRow& r, int k0, int keys) {
  const int n0 = max(k0 - r.context, -4096);  // key k0's node, negative in the context
  unsigned long long w;
  if (!p.mask) {
    const int c = r.node + 1 - n0;  // keys up to the row's own
    w = c >= 64 ? ~0ull : c <= 0 ? 0 : (1ull << c) - 1;
  } else {
    const int first = max(n0, 0) >> 6, sh = max(n0, 0) & 63;
    const unsigned long long* const m = p.mask + (long long)(r.q0 + max(r.node, 0)) * p.words + first;
    const unsigned long long a = first < p.words ? m[0] : 0, b = first + 1 < p.words ? m[1] : 0;
    w = sh ? a >> sh | b << (64 - sh) : a;
    if (n0 < 0) w = n0 <= -64 ? ~0ull : w << -n0 | ((1ull << -n0) - 1);
  }
  const int left = keys - k0;
  if (left < 64) w &= left <= 0 ? 0 : (1ull << left) - 1;
  return w;
}

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
template <class Params, int KEYS, int BLOCK, int WORKERS, int LEAD>
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
// A lane's query row of the block.
template <class L, class Params>
G9_DEV NodeRow row_of(const Params& p, const Place& at, int row) {
  const int nd = (at.block * L::kBlock + row) / p.group;
  const bool in = nd < at.r.n;
  return {in ? nd : -1, at.r.context, at.r.q0};
}
template <class L, class Params>
G9_DEV const char* query_of(const Params& p, const Place& at, int row, int node) {
  const int hd = at.block * L::kBlock + row - max(node, 0) * p.group;
  return p.q + (long long)(at.r.q0 + max(node, 0)) * p.q_t + (long long)(at.hk * p.group + (node < 0 ? 0 : hd)) * p.q_h;
}
// The row's results, or its sum to slot `slot` of the workspace.  o, m, l as the
// 32x32 layout leaves them: lane half h has the values 8 r + 4 h + 0..3 of every
// 32, l is its half of the weight.
template <bool BF16, int HD, class L, class Params>
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

// The joined row: with m the largest of the parts' maxima, the sum of 2^(m_i - m)
// O_i over the sum of 2^(m_i - m) l_i, in the order of the keys.
template <bool BF16, class Params>
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
constexpr int kJoinThreads = HD <= 128 ? 4 * HD : 512;
template <bool BF16, int HD, class L, class Params>
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

}  // namespace fa
}  // namespace g9
