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
constexpr int kLds = 4 * kTile;
constexpr float kNone = -3.0e38f;                // the maximum of a row that has read nothing: finite, weights 0

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

// One sum out of the accumulation registers (as assembly: the compiler would move all 16 of
// a block at once, and keep what it had in their place in scratch memory).
G9_DEV float sum_of(const f32x16& c, int i) {
  float x;
  asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(x) : "a"(c[i]));
  return x;
}

// The lane, worked out where it is used: what follows from it is not held through the loop.
G9_DEV int lane_here() {
  int x;
  asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(x));
  return x;
}

// RB blocks of 32 rows share a tile; a step of the workgroup is 4 / RB tiles.
template <int RB>
using Steps = Line<Params, kKeys * (4 / RB), 32 * RB, kWgs, 0>;

// One wave's rows and their sums.
template <bool BF16, int RB>
struct Rows {
  static constexpr int kGroups = 4 / RB;       // waves that take tiles in turn
  static constexpr int kPieces = 2;            // 16-row pieces of a tile: never across a page
  static constexpr int kDmas = 36 / RB;        // of a wave, for its group's tile

  const Params& p;
  u32 lds;             // of the workgroup
  u32 voff[9], flip;
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
    const int lane = threadIdx.x & 63, h = lane >> 5, col = lane & 31;
    lds = (u32)(uintptr_t)to_lds(smem);
    // Nine DMAs fill 8 rows: DMA j writes the bytes 1024 j + 16 lane of them.  The 8
    // rows behind them have bit 1 of their places the other way round: 32 bytes up or down.
    flip = 0;
#pragma unroll
    for (int j = 0; j < 9; ++j) {
      const int n = 64 * j + lane, r = n / 72, c = (n - 72 * r) ^ swz(r + (RB == 4 ? 8 * (wave & 1) : 0));
      voff[j] = (u32)r * p.c_t + 16 * c;
      flip |= (u32)(c >> 1 & 1) << j;
    }
    ak = col * kRowBytes + 16 * (h ^ swz(col));
    // 16 lanes cover 4 rows and 16 values: lane jj of them row jj / 4, values 4 (jj % 4)
    // of two pieces.
    const int jj = lane & 15, r4 = 4 * h + (jj >> 2);
    av = r4 * kRowBytes + 16 * ((2 * (lane >> 4 & 1) + ((jj & 3) >> 1)) ^ swz(r4)) + 8 * (jj & 1);
  }

  // This wave's share of the tile that begins with key k0, of `all` keys, into stage
  // `stage`; pg: the pages of the tile's two 16-row pieces.
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
      const u32 to = lds + stage * kTile + i * 16 * kRowBytes;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        if (RB == 4 && half != (wave & 1)) continue;
#pragma unroll
        for (int j = 0; j < 9; ++j) {
          const u32 at = RB == 4 || !half ? voff[j] : voff[j] + 32 - ((flip >> j & 1) << 6);
          dma16_fresh(r, to + 9216 * half + 1024 * j, at, half * 8 * p.c_t);
        }
      }
    }
  }

  G9_DEV void begin(const char* qrow) {
    const int h = lane_here() >> 5;
#pragma unroll
    for (int s = 0; s < kQk; ++s) qf[s] = *reinterpret_cast<const u32x4*>(qrow + (16 * s + 8 * h) * 2);
    m = kNone, l = 0.f;
#pragma unroll
    for (int d = 0; d < kPv; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float x;
        asm volatile("v_accvgpr_write_b32 %0, 0" : "=a"(x));
        o[d][i] = x;
      }
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
    u32x4 keep[2];  // TAIL: the keys whose values enter the product
    if constexpr (TAIL) {
      const int h = lane_here() >> 5;
      const u32 reads = (u32)node_reads(p, row, k0, keys), bad = special(stage);
      u32 quiet;  // a NaN that the compiler, told not to mind them, does not see
      asm("v_mov_b32 %0, 0x7fc00000" : "=v"(quiet));
      const u32 bits = reads >> (4 * h), nan = (reads & bad) >> (4 * h);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int key = 8 * (i / 4) + i % 4;
        const float x = __uint_as_float(nan >> key & 1 ? quiet : __float_as_uint(sc[i]));
        sc[i] = bits >> key & 1 ? x : -__builtin_inff();
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const u32 two = bad >> (4 * h + 16 * (i / 4) + 8 * (i / 2 % 2) + 2 * (i % 2));
        keep[i / 4][i % 4] = (two & 1 ? 0 : 0xffffu) | (two & 2 ? 0 : 0xffff0000u);
      }
    }
    float top = sc[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) top = __builtin_fmaxf(top, sc[i]);
    top = xhalf(top, [](float x, float y) { return __builtin_fmaxf(x, y); }) * p.scale_log2;
    const bool moves = top - m > kLazyThreshold;
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(moves) != 0, 0)) {
      const float m_new = moves ? top : m;
      const float alpha = __builtin_amdgcn_exp2f(m - m_new);
      const bool first = m < kNone * 0.5f;
      m = m_new;
      l *= alpha;
      // A row's first tile moves its maximum, but not its sums, which are zeros.
      if (__builtin_amdgcn_ballot_w64(moves && !first)) {
        settle(o);
#pragma unroll
        for (int d = 0; d < kPv; ++d) {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float x = o[d][i], y;
            asm volatile("v_accvgpr_read_b32 %1, %0\n\tv_mul_f32 %1, %1, %2\n\tv_accvgpr_write_b32 %0, %1"
                         : "+a"(x), "=&v"(y)
                         : "v"(alpha));
            o[d][i] = x;
          }
        }
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
#pragma unroll
    for (int i = 0; i < 2 * kPv; ++i) {
      // Block d of the sums, 16 of the keys at a time: fragment kQk + i.
      if constexpr (TAIL) {
        f[(kQk + i) % kDepth] &= keep[i / kPv];
        asm volatile("s_nop 1" : "+v"(f[(kQk + i) % kDepth]));
      }
      product<BF16>(o[i % kPv], f[(kQk + i) % kDepth], pf[i / kPv]);
      __builtin_amdgcn_sched_barrier(0);
      if (i + kDepth < 2 * kPv) f[(kQk + i) % kDepth] = v_at(i + kDepth);
    }
  }

  // The keys of the tile that hold an infinite or NaN latent.  A weight of 0 would not
  // keep such a value out of a row that does not read its key: where not every row
  // reads every key, these keys' values are left out of the product, and the rows that do
  // read one get a score of NaN (the latent is the key too: its product with the
  // query would be infinite or NaN).
  G9_DEV u32 special(int stage) const {
    typedef unsigned short h2 __attribute__((ext_vector_type(2)));
    constexpr u32 kExp = BF16 ? 0x7f80u : 0x7c00u;
    h2 top = {0, 0};
    const int lane = lane_here(), h = lane >> 5, col = lane & 31;
    // Half a latent a lane; the order of its pieces so that 16 rows touch every bank once.
    const u32 at = lds + stage * kTile + col * kRowBytes + 512 * h + 16 * (col >> 1 & 7);
#pragma unroll 8
    for (int j = 0; j < 32; ++j) {
      const u32x4 x = *(const G9_LDS u32x4*)(uintptr_t)((at ^ (16 * (j & 7))) + 128 * (j >> 3));
#pragma unroll
      for (int e = 0; e < 4; ++e) top = __builtin_elementwise_max(top, __builtin_bit_cast(h2, x[e] & 0x7fff7fffu));
    }
    const unsigned long long who = __builtin_amdgcn_ballot_w64(top.x >= kExp || top.y >= kExp);
    return (u32)who | (u32)(who >> 32);
  }
};

// A wave's results, or its sums to slot `slot` of the workspace, where no other wave
// has summed the same rows.  Branches of lanes are not nested: nothing may come between the
// ends of two of them.
template <bool BF16, int RB, class L>
G9_DEV void finish_rows(const Params& p, const Place& at, int slot, int in_block, const Rows<BF16, RB>& w) {
  const int h = lane_here() >> 5;
  const float l = xhalf(w.l, [](float x, float y) { return x + y; });
  const int node = w.row.node;
  if (slot >= 0) {
    const size_t to = (size_t)slot * L::kBlock + in_block;
    float* const sum = p.part + to * kRank + 4 * h;
    if (node >= 0) {
#pragma unroll
      for (int d = 0; d < kPv; ++d) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          *reinterpret_cast<f32x4*>(sum + 32 * d + 8 * r) =
              f32x4{w.o[d][4 * r], w.o[d][4 * r + 1], w.o[d][4 * r + 2], w.o[d][4 * r + 3]};
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if (node >= 0 && h == 0) {
      float* const ml = p.part + (size_t)2 * L::kWorkers * L::kBlock * kRank + to * 2;
      ml[0] = w.m, ml[1] = l;
    }
    return;
  }
  const int hq = at.block * L::kBlock + in_block - node * p.group;
  const long long tok = at.r.q0 + node;
  // By its bits: comparisons here may take NaN for a number.
  const bool none = (__float_as_uint(l) << 1) == 0;
  const float inv = none ? 0.f : 1.f / l;
  char* const orow = p.o + tok * p.o_t + hq * p.o_h + 8 * h;
  if (node >= 0) {
#pragma unroll
    for (int d = 0; d < kPv; ++d) {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        *reinterpret_cast<u32x2*>(orow + (32 * d + 8 * r) * 2) =
            u32x2{pack2<BF16>(sum_of(w.o[d], 4 * r) * inv, sum_of(w.o[d], 4 * r + 1) * inv),
                  pack2<BF16>(sum_of(w.o[d], 4 * r + 2) * inv, sum_of(w.o[d], 4 * r + 3) * inv)};
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  if (node >= 0 && h == 0 && p.lse)
    p.lse[(long long)hq * p.T + tok] = none ? -__builtin_inff() : (w.m + __builtin_log2f(l)) * kLn2;
}

// The waves of a block's groups have summed different keys of the same rows: joined in
// LDS, 256 of the 512 values at a time, and written as `finish` does.
template <bool BF16, int RB, class L>
G9_DEV void finish_groups(const Params& p, const Place& at, int slot, char* smem, int wave, const Rows<BF16, RB>& w) {
  constexpr int kGroups = 4 / RB, kPitch = 256 + 4, kSums = 32 * kPitch;  // 16 bytes more a row: banks
  static_assert((4 * kSums + 4 * 64) * 4 <= kLds);
  float* const sums = reinterpret_cast<float*>(smem);
  float* const ml = sums + 4 * kSums;  // maximum and weight of wave w's row r: [w][2][32]
  const int lane = lane_here(), h = lane >> 5, col = lane & 31;
  const float lw = xhalf(w.l, [](float x, float y) { return x + y; });
  barrier();  // every wave has read its tiles
  if (h == 0) ml[wave * 64 + col] = w.m, ml[wave * 64 + 32 + col] = lw;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    if (half) __syncthreads();
#pragma unroll
    for (int d = 0; d < 8; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const f32x16& x = w.o[8 * half + d];
        *reinterpret_cast<f32x4*>(sums + wave * kSums + col * kPitch + 32 * d + 8 * r + 4 * h) =
            f32x4{sum_of(x, 4 * r), sum_of(x, 4 * r + 1), sum_of(x, 4 * r + 2), sum_of(x, 4 * r + 3)};
        __builtin_amdgcn_sched_barrier(0);
      }
    __syncthreads();
    // A wave per row, 4 values a lane.
    for (int row = wave; row < 32 * RB; row += 4) {
      const int node = row_of<L>(p, at, row).node;
      if (node < 0) break;  // rows behind it neither
      const int rb = row >> 5, in = row & 31;
      float m = kNone, f[kGroups], l = 0.f;
#pragma unroll
      for (int g = 0; g < kGroups; ++g) m = __builtin_fmaxf(m, ml[(g * RB + rb) * 64 + in]);
      f32x4 x = {};
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        f[g] = __builtin_amdgcn_exp2f(ml[(g * RB + rb) * 64 + in] - m);
        l += f[g] * ml[(g * RB + rb) * 64 + 32 + in];
        x += f[g] * *reinterpret_cast<const f32x4*>(sums + (g * RB + rb) * kSums + in * kPitch + 4 * lane);
      }
      const int col = 256 * half + 4 * lane;
      if (slot >= 0) {
        *reinterpret_cast<f32x4*>(p.part + ((size_t)slot * L::kBlock + row) * kRank + col) = x;
        if (half == 0 && lane == 0) {
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
    const int in_block = 32 * (wave % RB) + (lane_here() & 31);
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
      finish_rows<BF16, RB, L>(p, cur, slot, in_block, w);
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
