// Attention over a paged cache of latents (g9_latent_fwd, include/gfx950_fmha.h):
// a token's row holds one latent of 512 values, which is every head's value and the
// larger part of its key, and a rotated key of 64 that the heads share too.
//
// All heads read the same row of 1152 bytes, for 2 (576 + 512) flops each: with 16
// heads the cache's bytes bound the call, with 128 (242 flops a byte) they still
// do by a little, if the products come near the matrix unit's rate.  So a row of the cache
// should reach a CU once for all its heads.
//
// The work is the line of g9_line.hpp, cut into one part per CU.  A workgroup is four
// waves, one per SIMD with the whole register file: a wave has 32 query rows, their
// sums of 512 values (256 accumulation registers a lane) and their queries (144
// registers).  RB = 1, 2 or 4 waves with different rows share each tile of 32 keys in
// LDS, and the 4 / RB groups take tiles in turn, whose sums are joined in LDS at the
// block's end.  Four tiles (147 KB) are in LDS, filled by LDS-DMA.
//
// Per tile a wave computes S^T = K Q^T and O^T += V^T P^T with 32x32x16 MFMAs, 36
// and 32 of them, in the register layouts that g9_fmha.hip describes: the weights
// P are rounded to the 16-bit type for that product (fp32 products have a sixteenth of the
// rate), their sum is taken before.  V is the row's first 512 values, read by
// transposing LDS reads.  A row's maximum moves only where a tile passes it by more
// than 8 (log2 units), so that the sums are rarely rescaled.
#include "../../include/gfx950_fmha.h"
#include "g9_attn_host.hpp"
#include "g9_line.hpp"

namespace g9 {
namespace latent {

using namespace fa;

constexpr int kRank = 512, kRow = 576;  // values of a latent, of a row
constexpr int kRowBytes = kRow * 2;
constexpr int kKeys = 32;               // of a tile
constexpr int kTile = kKeys * kRowBytes;
constexpr int kQk = kRow / 16, kPv = kRank / 32;  // products' steps of 16, blocks of 32 values
constexpr int kDepth = 6;                          // fragments read ahead
constexpr int kScratch = 32 * kKeys * 2;          // P of a wave's tile, 16 bit
constexpr int kLds = 4 * kTile + 4 * kScratch;

struct Params {
  const char* q;
  const char* cache;
  char* o;
  float* lse;                                      // [H][T], or null
  const int* table;
  const int* lengths;
  const int* cu;
  const unsigned long long* mask;                  // or null: a chain
  float* part;                                     // sums [2 kWgs][rows][512], then (m, l) pairs
  Start* start;                                    // [kWgs]: where each part begins
  long long q_t, q_h, o_t, o_h;                    // token / head strides, bytes
  long long c_b;                                   // block stride, bytes
  long long table_stride;
  u32 c_t;                                         // token stride, bytes
  int num_blocks, width, shift, words;
  int B, T, HK, group;                             // HK is 1, group the heads
  float scale_log2;
};

// The products as assembly, which keeps the sums in accumulation registers and the
// scores out of them.  The compiler does not look into it: the wait states between
// a product and the vector unit's use of its result, or of an operand that the vector unit
// has just written, are `settle` below (isa_check verifies them).
template <bool BF16>
G9_DEV void product(f32x16& c, u32x4 a, u32x4 b) {
  if constexpr (BF16)
    asm("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
  else
    asm("v_mfma_f32_32x32x16_f16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
}
template <bool BF16>
G9_DEV void score(f32x16& c, u32x4 a, u32x4 b) {
  if constexpr (BF16)
    asm("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+v"(c) : "v"(a), "v"(b));
  else
    asm("v_mfma_f32_32x32x16_f16 %0, %1, %2, %0" : "+v"(c) : "v"(a), "v"(b));
}
template <bool BF16>
G9_DEV void first_score(f32x16& c, u32x4 a, u32x4 b) {
  if constexpr (BF16)
    asm("v_mfma_f32_32x32x16_bf16 %0, %1, %2, 0" : "=&v"(c) : "v"(a), "v"(b));
  else
    asm("v_mfma_f32_32x32x16_f16 %0, %1, %2, 0" : "=&v"(c) : "v"(a), "v"(b));
}
G9_DEV void settle(f32x16& c) { asm volatile("s_nop 7\n\ts_nop 7" : "+v"(c)); }
G9_DEV void settle(f32x16 (&c)[kPv]) {
  asm volatile("s_nop 7\n\ts_nop 7" : "+a"(c[0]), "+a"(c[1]), "+a"(c[2]), "+a"(c[3]), "+a"(c[4]), "+a"(c[5]), "+a"(c[6]), "+a"(c[7]));
  asm volatile("" : "+a"(c[8]), "+a"(c[9]), "+a"(c[10]), "+a"(c[11]), "+a"(c[12]), "+a"(c[13]), "+a"(c[14]), "+a"(c[15]));
}
// Operands that the vector unit wrote, before the products that take them.
G9_DEV void ready(u32x4 (&x)[2]) { asm volatile("s_nop 1" : "+v"(x[0]), "+v"(x[1])); }

// RB blocks of 32 rows share a tile; a step of the workgroup is 4 / RB tiles.
template <int RB>
using Steps = Line<Params, kKeys * (4 / RB), 32 * RB, kWgs, 0>;

// One wave's rows and their sums.
template <bool BF16, int RB>
struct Rows {
  static constexpr int kGroups = 4 / RB;       // waves that take tiles in turn
  static constexpr int kPieces = 2;            // 16-row pieces of a tile: never across a page
  static constexpr int kDmas = 36 / RB;        // of a wave, for its group's tile
  static constexpr int kOffs = RB == 4 ? 9 : 18;  // different lane offsets of them

  const Params& p;
  int lane, h, col;
  u32 lds;             // of the workgroup
  char* scratch;
  u32 voff[kOffs];
  u32 ak, av;          // LDS read bases in a tile (K, V)
  u32x4 qf[kQk];
  f32x16 o[kPv];
  float m, l;
  NodeRow row;
  int keys;

  G9_DEV explicit Rows(const Params& pp) : p(pp) {}

  // A tile in LDS: rows of 1152 bytes (72 pieces of 16 bytes, an odd number of 128-byte
  // lines), piece c of row r at place c ^ swz(r).  A K read takes one piece of 16 rows:
  // (r & 1, swz(r)) is different for each, so it touches every bank once.  A
  // transposing V read takes 4 pieces of 4 rows: bit 2 of swz is bit 1 of r.
  static G9_DEV int swz(int r) { return (r >> 1 & 1) << 2 | (r >> 2 & 3); }

  G9_DEV void init(char* smem, int wave) {
    lane = threadIdx.x & 63, h = lane >> 5, col = lane & 31;
    lds = (u32)(uintptr_t)to_lds(smem);
    scratch = smem + 4 * kTile + wave * kScratch;
    // DMA j of a 16-row piece writes its bytes 1024 j + 16 lane.
#pragma unroll
    for (int j = 0; j < kOffs; ++j) {
      const int n = 64 * (j + (RB == 4 ? 9 * (wave & 1) : 0)) + lane, r = n / 72, place = n - 72 * r;
      voff[j] = (u32)r * p.c_t + 16 * (place ^ swz(r));
    }
    ak = col * kRowBytes + 16 * (h ^ swz(col));
    // 16 lanes cover 4 rows and 16 values: lane jj of them row jj / 4, values 4 (jj % 4)
    // of two pieces.
    const int jj = lane & 15, r4 = 4 * h + (jj >> 2);
    av = r4 * kRowBytes + 16 * ((2 * (lane >> 4 & 1) + ((jj & 3) >> 1)) ^ swz(r4)) + 8 * (jj & 1);
  }

  // This wave's share of the tile that begins with key k0 of request b, into stage
  // `stage`: pieces by = the pages of its two 16-row pieces.
  G9_DEV void fill(int stage, int k0, int all, const int (&pg)[kPieces], int wave) const {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      if (RB == 4 && i != wave >> 1) continue;
      if (RB == 2 && i != (wave & 1)) continue;
      const int k = k0 + 16 * i, off = k & ((1 << p.shift) - 1);
      const bool in = (u32)pg[i] < (u32)p.num_blocks;
      const int rows = in ? min(max(all - k, 0), 16) : 0;
      const char* const base = p.cache + (long long)(in ? pg[i] : 0) * p.c_b + (unsigned long long)(u32)off * p.c_t;
      const rsrc_t r = make_rsrc(uniform(base), uniform(extent(rows, p.c_t, kRowBytes)));
      const u32 to = lds + stage * kTile + i * 16 * kRowBytes + (RB == 4 ? 9 * 1024 * (wave & 1) : 0);
#pragma unroll
      for (int j = 0; j < kOffs; ++j) dma16_fresh(r, to + 1024 * j, voff[j], 0);
    }
  }

  G9_DEV void begin(const char* qrow) {
#pragma unroll
    for (int s = 0; s < kQk; ++s) qf[s] = *reinterpret_cast<const u32x4*>(qrow + (16 * s + 8 * h) * 2);
    m = -3.0e38f, l = 0.f;  // finite: a row that has read nothing has weights of 0
#pragma unroll
    for (int d = 0; d < kPv; ++d) o[d] = f32x16{};
  }

  G9_DEV u32x4 v_at(u32 base, int k, int d) const {
    const u32 a = (base ^ (64 * (d & 1))) + 128 * (d >> 1) + 16 * kRowBytes * k;
    const u32 b = (base ^ (64 * (d & 1) + 32)) + 128 * (d >> 1) + 16 * kRowBytes * k + 8 * kRowBytes;
    const u32x2 lo = tr_read(a), hi = tr_read(b);
    return u32x4{lo.x, lo.y, hi.x, hi.y};
  }

  // Adds the tile in `stage`, whose first key is k0; TAIL: not every row may read all of it.
  template <bool TAIL>
  G9_DEV void tile(int k0, int stage) {
    const u32 ks = lds + stage * kTile + ak, vs = lds + stage * kTile + av;
    // Fragments are read kDepth ahead of the product that takes them (the compiler takes
    // assembly for instructions without a latency, and would read each just before).
    const u32 kb[4] = {ks, ks ^ 32, ks ^ 64, ks ^ 96}, vb[4] = {vs, vs ^ 64, vs ^ 32, vs ^ 96};
    const auto k_at = [&](int s) { return *(const G9_LDS u32x4*)(uintptr_t)(kb[s & 3] + 128 * (s >> 2)); };
    const auto v_at = [&](int i) {
      const int at = 16 * kRowBytes * (i / kPv) + 128 * (i % kPv >> 1);
      const u32x2 lo = tr_read(vb[i & 1] + at), hi = tr_read(vb[2 + (i & 1)] + at + 8 * kRowBytes);
      return u32x4{lo.x, lo.y, hi.x, hi.y};
    };
    u32x4 f[kDepth];
    f32x16 sc;
#pragma unroll
    for (int s = 0; s < kDepth; ++s) f[s] = k_at(s);
#pragma unroll
    for (int s = 0; s < kQk; ++s) {
      if (s == 0)
        first_score<BF16>(sc, f[0], qf[0]);
      else
        score<BF16>(sc, f[s % kDepth], qf[s]);
      __builtin_amdgcn_sched_barrier(0);
      f[s % kDepth] = s + kDepth < kQk ? k_at(s + kDepth) : v_at(s + kDepth - kQk);
    }
    settle(sc);
    if constexpr (TAIL) {
      const u32 bits = (u32)node_reads(p, row, k0, keys) >> (4 * h);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float x = sc[i];
        sc[i] = bits >> (8 * (i / 4) + i % 4) & 1 ? x : -__builtin_inff();
      }
    }
    float top = sc[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) top = __builtin_fmaxf(top, sc[i]);
    top = xhalf(top, [](float x, float y) { return __builtin_fmaxf(x, y); }) * p.scale_log2;
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(top - m > kLazyThreshold) != 0, 0)) {
      const float m_new = top - m > kLazyThreshold ? top : m;
      const float alpha = __builtin_amdgcn_exp2f(m - m_new);
      m = m_new;
      l *= alpha;
      settle(o);
#pragma unroll
      for (int d = 0; d < kPv; ++d) {
        o[d] *= alpha;
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    u32x4 pf[2];
    float sum[4] = {};
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
      const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[i], p.scale_log2, -m));
      const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[i + 1], p.scale_log2, -m));
      sum[i / 2 % 2 * 2] += x, sum[i / 2 % 2 * 2 + 1] += y;
      pf[i / 8][i % 8 / 2] = pack2<BF16>(x, y);
    }
    l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
    ready(pf);
    if constexpr (TAIL)
      if (has_special(stage)) {
        special(k0, stage, pf);
        return;
      }
#pragma unroll
    for (int i = 0; i < 2 * kPv; ++i) {
      // Block d of the sums, 16 of the keys at a time: fragment kQk + i.
      product<BF16>(o[i % kPv], f[(kQk + i) % kDepth], pf[i / kPv]);
      __builtin_amdgcn_sched_barrier(0);
      if (i + kDepth < 2 * kPv) f[(kQk + i) % kDepth] = v_at(i + kDepth);
    }
  }

  static constexpr u32 kExp = BF16 ? 0x7f80u : 0x7c00u;
  // Whether a latent of the tile is infinite or NaN.
  G9_DEV bool has_special(int stage) const {
    typedef unsigned short h2 __attribute__((ext_vector_type(2)));
    h2 top = {0, 0};
    // Every piece, the rotated keys' too.
#pragma unroll 4
    for (int j = 0; j < kTile / 1024; ++j) {
      const u32x4 x = *(const G9_LDS u32x4*)(uintptr_t)(lds + stage * kTile + 1024 * j + 16 * lane);
#pragma unroll
      for (int e = 0; e < 4; ++e) top = __builtin_elementwise_max(top, __builtin_bit_cast(h2, x[e] & 0x7fff7fffu));
    }
    return __builtin_expect(__builtin_amdgcn_ballot_w64(top.x >= kExp || top.y >= kExp) != 0, 0);
  }
  // Such a tile, where not every row reads every key: a weight of 0 does not keep an
  // infinite or NaN value out of the product.  It is taken out there, and added on the
  // vector unit to the rows that read its key; all other sums keep their bits.
  G9_DEV void special(int k0, int stage, const u32x4 (&pf)[2]) {
    const u32 vs = lds + stage * kTile + av;
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int d = 0; d < kPv; ++d) {
        u32x4 v = v_at(vs, k, d);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if ((v[e] & kExp) == kExp) v[e] &= 0xffff0000u;
          if (((v[e] >> 16) & kExp) == kExp) v[e] &= 0xffffu;
        }
        asm volatile("s_nop 1" : "+v"(v));
        product<BF16>(o[d], v, pf[k]);
        __builtin_amdgcn_sched_barrier(0);
      }
    settle(o);
    // P in LDS: row of the query, column of the key.
    uint16_t* const prow = reinterpret_cast<uint16_t*>(scratch) + col * kKeys;
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) *reinterpret_cast<u32*>(prow + 16 * k + 8 * (e >> 1) + 4 * h + 2 * (e & 1)) = pf[k][e];
    const u32 reads = (u32)node_reads(p, row, k0, keys);
    waitcnt<63, 0>();
#pragma unroll 1
    for (int key = 0; key < kKeys; ++key) {
      if (!(reads >> key & 1)) continue;
      const float w = unpack2<BF16>(prow[key]).x;
      const u32 vr = lds + stage * kTile + key * kRowBytes + 8 * h;
      const u32 sw = swz(key);
#pragma unroll
      for (int d = 0; d < kPv; ++d)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const u32x2 x = *(const G9_LDS u32x2*)(uintptr_t)(vr + 16 * ((4 * d + r) ^ sw));
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            u32 y = (e & 1 ? x[e / 2] >> 16 : x[e / 2]) & 0xffffu;
            if ((y & kExp) != kExp) y = 0;
            o[d][4 * r + e] += w * unpack2<BF16>(y).x;
          }
          __builtin_amdgcn_sched_barrier(0);
        }
    }
  }
};

// The waves of a block's groups have summed different keys of the same rows: joined in
// LDS, 256 of the 512 values at a time, and written as `finish` does.
template <bool BF16, int RB, class L>
G9_DEV void finish_groups(const Params& p, const Place& at, int slot, char* smem, int wave, const Rows<BF16, RB>& w) {
  constexpr int kGroups = 4 / RB, kPitch = 256 + 4, kSums = 32 * kPitch;  // 16 bytes more a row: banks
  static_assert((4 * kSums + 4 * 64) * 4 <= kLds);
  float* const sums = reinterpret_cast<float*>(smem);
  float* const ml = sums + 4 * kSums;  // maximum and weight of wave w's row r: [w][2][32]
  const float lw = xhalf(w.l, [](float x, float y) { return x + y; });
  barrier();  // every wave has read its tiles
  if (w.h == 0) ml[wave * 64 + w.col] = w.m, ml[wave * 64 + 32 + w.col] = lw;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    if (half) __syncthreads();
#pragma unroll
    for (int d = 0; d < 8; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const f32x16& x = w.o[8 * half + d];
        *reinterpret_cast<f32x4*>(sums + wave * kSums + w.col * kPitch + 32 * d + 8 * r + 4 * w.h) =
            f32x4{x[4 * r], x[4 * r + 1], x[4 * r + 2], x[4 * r + 3]};
      }
    __syncthreads();
    // A wave per row, 4 values a lane.
    for (int row = wave; row < 32 * RB; row += 4) {
      const int node = row_of<L>(p, at, row).node;
      if (node < 0) break;  // rows behind it neither
      const int rb = row >> 5, in = row & 31;
      float m = -3.0e38f, f[kGroups], l = 0.f;
#pragma unroll
      for (int g = 0; g < kGroups; ++g) m = __builtin_fmaxf(m, ml[(g * RB + rb) * 64 + in]);
      f32x4 x = {};
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        f[g] = __builtin_amdgcn_exp2f(ml[(g * RB + rb) * 64 + in] - m);
        l += f[g] * ml[(g * RB + rb) * 64 + 32 + in];
        x += f[g] * *reinterpret_cast<const f32x4*>(sums + (g * RB + rb) * kSums + in * kPitch + 4 * w.lane);
      }
      const int col = 256 * half + 4 * w.lane;
      if (slot >= 0) {
        *reinterpret_cast<f32x4*>(p.part + ((size_t)slot * L::kBlock + row) * kRank + col) = x;
        if (half == 0 && w.lane == 0) {
          float* const to = p.part + (size_t)2 * L::kWorkers * L::kBlock * kRank + ((size_t)slot * L::kBlock + row) * 2;
          to[0] = m, to[1] = l;
        }
      } else {
        const int hq = at.block * L::kBlock + row - node * p.group;
        store4<BF16>(p, at.r.q0 + node, hq, col / 4, x, m, l);
      }
    }
  }
  __syncthreads();  // the next block's tiles take the sums' place
}

template <bool BF16, int RB>
G9_DEV void fwd(const Params& p, char* smem) {
  using L = Steps<RB>;
  using R = Rows<BF16, RB>;
  constexpr int kGroups = R::kGroups, kAhead = RB - 1;  // steps asked for ahead: the stages of a group but one
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int group = wave / RB;
  const unsigned worker = my_part();
  Place cur{};
  int left = L::template locate<256>(p, smem, worker, cur);
  R w(p);
  w.init(smem, wave);
  while (left > 0) {
    const int seg = min(left, cur.r.tiles - cur.tile);
    const bool last = cur.tile + seg == cur.r.tiles, from_start = cur.tile == 0;
    const int first = cur.tile * L::kKeys + group * kKeys;  // this wave's first key
    const int in_block = 32 * (wave % RB) + w.col;
    w.row = row_of<L>(p, cur, in_block);
    w.keys = cur.r.keys;
    const int* const table = p.table + cur.b * p.table_stride;
    const auto pages = [&](int step, int (&pg)[2]) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int k = first + step * L::kKeys + 16 * i;
        pg[i] = k < cur.r.keys ? table[k >> p.shift] : -1;
      }
    };
    const auto ask = [&](int step, const int (&pg)[2]) {
      w.fill(group * RB + step % RB, first + step * L::kKeys, cur.r.keys, pg, wave);
    };
    int pg[2];
#pragma unroll
    for (int i = 0; i < (kAhead ? kAhead : 1); ++i)
      if (i < seg) {
        pages(i, pg);
        ask(i, pg);
      }
    const int next = kAhead ? kAhead : 1;
    if (next < seg) pages(next, pg);
    w.begin(query_of<L>(p, cur, in_block, w.row.node));
    waitcnt<0, 0>();
    // Rows of this wave, tiles that none of them reads.
    const bool some = cur.block * L::kBlock + 32 * (wave % RB) < cur.r.n * p.group;
    const int whole = min(cur.r.context, cur.r.keys);  // keys that every row reads
    const auto steps = [&]<bool TAIL>(int from, int to) {
#pragma unroll 1
      for (int j = from; j < to; ++j) {
          if constexpr (RB > 1) {
            // Step j has landed (steps up to j + kAhead - 1 are asked for), for every wave of the group.
            if (kAhead > 2 && j + 2 < seg)
              waitcnt<2 * R::kDmas, 15>();
            else if (kAhead > 1 && j + 1 < seg)
              waitcnt<R::kDmas, 15>();
            else
              waitcnt<0, 15>();
            barrier();
            if (j + kAhead < seg) {
              ask(j + kAhead, pg);
              if (j + kAhead + 1 < seg) pages(j + kAhead + 1, pg);
            }
          } else {
            waitcnt<0, 15>();
            __builtin_amdgcn_sched_barrier(0);
          }
          const int k0 = first + j * L::kKeys;
          if (some) w.template tile<TAIL>(k0, group * RB + j % RB);
          if constexpr (RB == 1) {
            waitcnt<63, 0>();
            __builtin_amdgcn_sched_barrier(0);
            if (j + 1 < seg) {
              ask(j + 1, pg);
              if (j + 2 < seg) pages(j + 2, pg);
            }
          }
      }
    };
    // The steps whose tiles every row reads whole, then the others.
    const int mid = min(max((whole - cur.tile * L::kKeys) / L::kKeys, 0), seg);
    steps.template operator()<false>(0, mid);
    steps.template operator()<true>(mid, seg);
    settle(w.o);
    const int slot = last && from_start ? -1 : (int)(2 * worker + (from_start ? 1 : 0));
    if constexpr (kGroups == 1) {
      finish<BF16, kRank, L>(p, cur, slot, in_block, w.row.node, w.o, w.m, w.l);
      barrier();  // the stages are read: the next block's tiles take them
    } else {
      finish_groups<BF16, RB, L>(p, cur, slot, smem, wave, w);
    }
    left -= seg + L::kLead;
    if (left > 0) cur = L::next_block(p, cur);
  }
}

}  // namespace latent
}  // namespace g9

using namespace g9;
using namespace g9::host;

#define G9_LATENT_KERNEL(NAME, BF16, RB)                                                                           \
  extern "C" __global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1, 1))) void                    \
  g9_latent_##NAME(latent::Params p) {                                                                            \
    __shared__ __attribute__((aligned(1024))) char smem[latent::kLds];                                            \
    latent::fwd<BF16, RB>(p, smem);                                                                               \
  }                                                                                                               \
  extern "C" __global__ __launch_bounds__(fa::kJoinThreads<512>) void g9_latent_join_##NAME(latent::Params p) {   \
    __shared__ float lds[fa::kJoinThreads<512> * 7];                                                              \
    fa::join<BF16, 512, latent::Steps<RB>>(p, lds);                                                               \
  }
G9_LATENT_KERNEL(bf16_q32, true, 1)
G9_LATENT_KERNEL(f16_q32, false, 1)
G9_LATENT_KERNEL(bf16_q64, true, 2)
G9_LATENT_KERNEL(f16_q64, false, 2)
G9_LATENT_KERNEL(bf16_q128, true, 4)
G9_LATENT_KERNEL(f16_q128, false, 4)

namespace {

// Query rows of a block, by the rows (nodes by heads) that a request of the batch
// brings on average.
enum { Q32, Q64, Q128 };
int form_of(int64_t B, int64_t T, int64_t H) {
  const int64_t rows = (T + B - 1) / B * H;
  return rows <= 32 ? Q32 : rows <= 64 ? Q64 : Q128;
}
// The workspace: the sums of 2 x 256 blocks and their (m, l) pairs, then start[].
size_t start_at(int form) { return (size_t)2 * fa::kWgs * (32 << form) * (512 + 2) * 4; }

#define G9_LATENT_FN(WHAT, Q) {reinterpret_cast<const void*>(WHAT##f16_##Q), reinterpret_cast<const void*>(WHAT##bf16_##Q)}
const void* const kRun[3][2] = {G9_LATENT_FN(g9_latent_, q32), G9_LATENT_FN(g9_latent_, q64), G9_LATENT_FN(g9_latent_, q128)};
const void* const kJoin[3][2] = {G9_LATENT_FN(g9_latent_join_, q32), G9_LATENT_FN(g9_latent_join_, q64),
                                 G9_LATENT_FN(g9_latent_join_, q128)};

}  // namespace

extern "C" size_t g9_latent_workspace_size(int64_t B, int64_t T, int64_t H) {
  if (B <= 0 || T <= 0 || H <= 0) return 0;
  return start_at(form_of(B, T, H)) + fa::kWgs * sizeof(fa::Start);
}

extern "C" int g9_latent_fwd(const void* q, const void* cache, void* o, float* lse, const int32_t* block_table,
                             int64_t table_stride, int64_t width, const int32_t* lengths, const int32_t* cu_q,
                             const int64_t* tree_mask, int64_t words, int64_t B, int64_t T, int64_t H,
                             int64_t num_blocks, int64_t block_size, const int64_t* q_strides,
                             const int64_t* cache_strides, const int64_t* o_strides, float sm_scale, int dtype,
                             void* workspace, size_t workspace_bytes, void* stream) {
  using latent::kRank, latent::kRow;
  if (dtype != G9_F16 && dtype != G9_BF16) return G9_ERR_DTYPE;
  if (B < 0 || B > G9_TREE_MAX_REQUESTS || T < 0 || T > kMaxRows || H <= 0 || H > 65536 || !scale_ok(sm_scale) ||
      num_blocks < 0 || num_blocks > kMaxRows || width < 0 || width > kMaxRows || !block_size_ok(block_size) ||
      width * block_size > (int64_t(1) << 30) || words < 0 || words > 1024 || (tree_mask && words == 0))
    return G9_ERR_SHAPE;
  if (!q_strides || !cache_strides || !o_strides) return G9_ERR_LAYOUT;
  // The step of a single row is never taken.
  const int64_t qs[2] = {T > 1 ? q_strides[0] : 0, H > 1 ? q_strides[1] : 0};
  const int64_t os[2] = {T > 1 ? o_strides[0] : 0, H > 1 ? o_strides[1] : 0};
  const int64_t cs[2] = {num_blocks > 1 ? cache_strides[0] : 0, cache_strides[1]};
  if (!steps(qs, 2) || !steps(cs, 2) || !steps(os, 2)) return G9_ERR_LAYOUT;
  const int64_t size[2] = {T, H};
  if (!apart(size, os, 2, kRank) || (B > 1 && table_stride < width)) return G9_ERR_LAYOUT;
  // A 16-row piece of a page lies within a descriptor's range, its rows apart.
  if (cs[1] < kRow || cs[1] * 2 * 16 >= (int64_t(1) << 31)) return G9_ERR_LAYOUT;
  if (T * H > INT32_MAX) return G9_ERR_SHAPE;
  if (B == 0 || T == 0) return G9_OK;
  if (!q || !o || !lengths || !cu_q || (width && !block_table) || (num_blocks && !cache)) return G9_ERR_LAYOUT;
  if (!aligned16(q) || !aligned16(cache) || !aligned16(o) || ((uintptr_t)lse & 3) || ((uintptr_t)tree_mask & 7))
    return G9_ERR_LAYOUT;
  const int form = form_of(B, T, H);
  if (!workspace || ((uintptr_t)workspace & 31) || workspace_bytes < g9_latent_workspace_size(B, T, H))
    return G9_ERR_WORKSPACE;
  latent::Params p{};
  p.q = static_cast<const char*>(q);
  p.cache = static_cast<const char*>(cache);
  p.o = static_cast<char*>(o);
  p.lse = lse;
  p.table = block_table;
  p.lengths = lengths;
  p.cu = cu_q;
  p.mask = reinterpret_cast<const unsigned long long*>(tree_mask);
  p.part = static_cast<float*>(workspace);
  p.start = reinterpret_cast<fa::Start*>(static_cast<char*>(workspace) + start_at(form));
  p.q_t = qs[0] * 2, p.q_h = qs[1] * 2, p.o_t = os[0] * 2, p.o_h = os[1] * 2;
  p.c_b = cs[0] * 2, p.c_t = (u32)(cs[1] * 2);
  p.table_stride = table_stride;
  p.num_blocks = (int)num_blocks, p.width = (int)width, p.shift = log2_of(block_size), p.words = (int)words;
  p.B = (int)B, p.T = (int)T, p.HK = 1, p.group = (int)H;
  p.scale_log2 = sm_scale * fa::kLog2e;
  void* args[] = {&p};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const int bf16 = dtype == G9_BF16;
  if (hipLaunchKernel(kRun[form][bf16], dim3(fa::kWgs), dim3(256), args, 0, st) != hipSuccess) return G9_ERR_HIP;
  return launched(hipLaunchKernel(kJoin[form][bf16], dim3(fa::kWgs - 1, form == Q128 ? 4 : 1),
                                  dim3(fa::kJoinThreads<512>), args, 0, st));
}
