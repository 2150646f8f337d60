// The work of the attentions over a paged cache (g9_tree.hip, g9_latent.hip) as a
// line of key tiles, cut into equal parts: which tiles a worker takes follows from
// the requests' lengths alone, and every worker finds its part itself.  And which keys
// a query row reads.
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

// Consecutive workgroups go round the 8 XCDs; consecutive parts of the line stay
// on one, whose L2 then serves the blocks of rows that share keys.
G9_DEV unsigned my_part() { return (blockIdx.x & 7) * (kWgs / 8) + (blockIdx.x >> 3); }

}  // namespace fa
}  // namespace g9
