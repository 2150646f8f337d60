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
  float* part;                                     // sums of 2 kWgs blocks (part_at), then (m, l) pairs
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
using Steps = Line<Params, kKeys * (4 / RB), 32 * RB, kWgs, RB == 4 ? 5 : 2>;

// One wave's rows and their sums.
template <bool BF16, int RB>
struct Rows {
  static constexpr int kGroups = 4 / RB;       // waves that take tiles in turn

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

  // A 16-row piece of a tile to come: its rows' descriptor, its place in LDS.
  struct Piece {
    rsrc_t r;
    u32 to;
  };
  // Piece i of the tile that begins with key k0, of `all` keys (rows behind them read as
  // zeros), on page pg, into stage `stage`.
  G9_DEV Piece aim(int i, int stage, int k0, int all, int pg) const {
    const int k = k0 + 16 * i, off = k & ((1 << p.shift) - 1);
    const bool in = (u32)pg < (u32)p.num_blocks;
    const int rows = in ? min(max(all - k, 0), 16) : 0;
    const char* const base = p.cache + (long long)(in ? pg : 0) * p.c_b + (unsigned long long)(u32)off * p.c_t;
    return {make_rsrc(uniform(base), uniform(extent(rows, p.c_t, kRowBytes))),
            (u32)uniform((int)(lds + stage * kTile + i * 16 * kRowBytes))};
  }
  // DMA j of a piece's 18.
  template <int J>
  G9_DEV void fetch(const Piece& x, int wave) const {
    if constexpr (RB == 4) {  // a wave has one half of a piece
      dma16_fresh(x.r, x.to + 9216 * (wave & 1) + 1024 * J, voff[J], (wave & 1) * 8 * p.c_t);
    } else {
      const u32 at = J < 9 ? voff[J % 9] : voff[J % 9] + 32 - ((flip >> (J % 9) & 1) << 6);
      dma16_fresh(x.r, x.to + 1024 * J, at, J < 9 ? 0 : 8 * p.c_t);
    }
  }
  static constexpr int kOwn = RB == 4 ? 9 : 18;  // a wave's DMAs of a piece
  template <int J = 0>
  G9_DEV void fetch_all(const Piece& x, int wave) const {
    if constexpr (J < kOwn) {
      fetch<J>(x, wave);
      fetch_all<J + 1>(x, wave);
    }
  }

  G9_DEV void load_q(const char* qrow) {
    const int h = lane_here() >> 5;
#pragma unroll
    for (int s = 0; s < kQk; ++s) qf[s] = *reinterpret_cast<const u32x4*>(qrow + (16 * s + 8 * h) * 2);
  }
  G9_DEV void clear() {
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
  // The DMAs of piece `next` (RB > 1) are issued between the products: all at once, they
  // would hold the wave until memory has taken them.
  template <bool TAIL>
  G9_DEV void tile(int k0, int stage, const Piece& next, int wave) {
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
    // DMA J behind product (2 J + 1) / 2 / kOwn of all.
    const auto slot = [&]<int S>() {
      constexpr int kAll = kQk + 2 * kPv, J = (2 * S + 1) * kOwn / (2 * kAll), K = (2 * S + 3) * kOwn / (2 * kAll);
      if constexpr (RB > 1 && J != K && J < kOwn) fetch<J>(next, wave);
    };
    f32x16 sc;
#pragma unroll
    for (int s = 0; s < kDepth; ++s) f[s] = k_at(s);
    const auto qk_step = [&]<int S>(auto self) {
      if constexpr (S < kQk) {
        if constexpr (S == 0)
          first_score<BF16>(sc, f[0], qf[0]);
        else
          score<BF16>(sc, f[S % kDepth], qf[S]);
        __builtin_amdgcn_sched_barrier(0);
        f[S % kDepth] = S + kDepth < kQk ? k_at(S + kDepth) : v_at(S + kDepth - kQk);
        slot.template operator()<S>();
        self.template operator()<S + 1>(self);
      }
    };
    qk_step.template operator()<0>(qk_step);
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
    const auto pv_step = [&]<int I>(auto self) {
      if constexpr (I < 2 * kPv) {
        // Block d of the sums, 16 of the keys at a time: fragment kQk + I.
        u32x4& v = f[(kQk + I) % kDepth];
        if constexpr (TAIL) {
          v &= keep[I / kPv];
          asm volatile("s_nop 1" : "+v"(v));
        }
        product<BF16>(o[I % kPv], v, pf[I / kPv]);
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (I + kDepth < 2 * kPv) v = v_at(I + kDepth);
        slot.template operator()<kQk + I>();
        self.template operator()<I + 1>(self);
      }
    };
    pv_step.template operator()<0>(pv_step);
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

// Sums in the workspace: [slot][32 rows][64 groups of 8 values][lane][4], as the products
// leave them, a lane being a row and half of the 8 values: whole lines, written and read.
template <int RB>
G9_DEV size_t part_at(size_t slot, int rb, int q) {
  return (((slot * RB + rb) * 64 + q) * 64) * 4;
}
template <int RB>
G9_DEV size_t ml_at(size_t slot, int row) {
  return (size_t)2 * kWgs * 32 * RB * kRank + (slot * 32 * RB + row) * 2;
}
// Where a lane's row goes: row `in` of the block.
struct Out {
  char* o;
  float* lse;
};
template <class P>
G9_DEV Out out_of(const P& p, int q0, int row, int node) {
  const int hq = row - node * p.group;
  const long long tok = q0 + node;
  return {p.o + tok * p.o_t + hq * p.o_h, p.lse ? p.lse + (long long)hq * p.T + tok : nullptr};
}
template <bool BF16>
G9_DEV u32x2 scaled(f32x4 x, float inv) {
  return u32x2{pack2<BF16>(x[0] * inv, x[1] * inv), pack2<BF16>(x[2] * inv, x[3] * inv)};
}
// By its bits: comparisons here may take NaN for a number.
G9_DEV bool nothing(float l) { return (__float_as_uint(l) << 1) == 0; }
G9_DEV float lse_of(float m, float l) { return nothing(l) ? -__builtin_inff() : (m + __builtin_log2f(l)) * kLn2; }

// A block's results, or its sums to slot `slot` of the workspace.  The groups' sums of the
// same rows (over different keys) are joined in LDS, 256 of the 512 values at a time; every
// wave takes a share of the values.  Branches of lanes are not nested: nothing may come
// between the ends of two of them.
template <bool BF16, int RB, class L>
G9_DEV void finish_block(const Params& p, const Place& at, int slot, char* smem, int wave, const Rows<BF16, RB>& w) {
  constexpr int kGroups = 4 / RB, kPitch = 256 + 4, kSums = 32 * kPitch;  // 16 bytes more a row: banks
  static_assert((4 * kSums + 4 * 64) * 4 <= kLds);
  const int lane = lane_here(), h = lane >> 5, col = lane & 31;
  float* const sums = reinterpret_cast<float*>(smem);
  float* const ml = sums + 4 * kSums;  // maximum and weight of wave w's row r: [w][2][32]
  const int rb = wave % RB, row = at.block * L::kBlock + 32 * rb + col, node = w.row.node;
  float m = w.m, l = xhalf(w.l, [](float x, float y) { return x + y; }), f[kGroups];
  waitcnt<0, 15>();  // the DMAs behind the last step
  barrier();         // every wave has read its tiles
  if constexpr (kGroups > 1) {
    if (h == 0) ml[wave * 64 + col] = m, ml[wave * 64 + 32 + col] = l;
    __syncthreads();
#pragma unroll
    for (int g = 0; g < kGroups; ++g) m = __builtin_fmaxf(m, ml[(g * RB + rb) * 64 + col]);
    l = 0.f;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      f[g] = __builtin_amdgcn_exp2f(ml[(g * RB + rb) * 64 + col] - m);
      l += f[g] * ml[(g * RB + rb) * 64 + 32 + col];
    }
  }
  const float inv = nothing(l) ? 0.f : 1.f / l;
  const Out out = out_of(p, at.r.q0, row, max(node, 0));
  const auto put = [&](int q, f32x4 x) {
    if (slot >= 0)
      *reinterpret_cast<f32x4*>(p.part + part_at<RB>(slot, rb, q) + 4 * lane) = x;
    else if (node >= 0)
      *reinterpret_cast<u32x2*>(out.o + 16 * q + 8 * h) = scaled<BF16>(x, inv);
  };
  const auto quad = [&](int q) {
    const f32x16& x = w.o[q / 4];
    const int r = 4 * (q % 4);
    return f32x4{sum_of(x, r), sum_of(x, r + 1), sum_of(x, r + 2), sum_of(x, r + 3)};
  };
  if constexpr (kGroups == 1) {
    if (slot >= 0) {
#pragma unroll
      for (int q = 0; q < 64; ++q) {
        put(q, quad(q));
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
#pragma unroll
      for (int q = 0; q < 64; ++q) {
        put(q, quad(q));
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  } else {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      if (half) __syncthreads();
#pragma unroll
      for (int q = 0; q < 32; ++q) {
        *reinterpret_cast<f32x4*>(sums + wave * kSums + col * kPitch + 8 * q + 4 * h) = quad(32 * half + q);
        __builtin_amdgcn_sched_barrier(0);
      }
      __syncthreads();
#pragma unroll 4
      for (int i = 0; i < 32 / kGroups; ++i) {
        const int q = wave / RB * (32 / kGroups) + i;
        f32x4 x = {};
#pragma unroll
        for (int g = 0; g < kGroups; ++g)
          x += f[g] * *reinterpret_cast<const f32x4*>(sums + (g * RB + rb) * kSums + col * kPitch + 8 * q + 4 * h);
        put(32 * half + q, x);
      }
    }
    __syncthreads();  // the next block's tiles take the sums' place
  }
  if (wave / RB == 0) {
    if (slot >= 0) {
      if (h == 0) *reinterpret_cast<f32x2*>(p.part + ml_at<RB>(slot, 32 * rb + col)) = f32x2{m, l};
    } else {
      if (h == 0 && node >= 0 && out.lse) *out.lse = lse_of(m, l);
    }
  }
}

// Joins the blocks that are cut.  A block of n parts has the n - 1 workers whose parts
// begin within it, and with each of them gridDim.y workgroups here, which share its groups
// of 32 rows by 8 values: a wave each where the parts are few, else a workgroup, whose
// waves share the parts.  In the order of the keys: with m the largest of the parts'
// maxima, the sum of 2^(m_i - m) O_i over the sum of 2^(m_i - m) l_i.
constexpr int kJoinWaves = 8, kFewParts = 8, kJoinUnits = 4;
constexpr int kJoinLds = kJoinWaves * 64 * (4 * kJoinUnits + 2);
template <bool BF16, int RB>
G9_DEV void join_parts(const Params& p, float* lds) {
  using L = Steps<RB>;
  const unsigned w = blockIdx.x + 1;
  const Start zero = p.start[0];
  const unsigned long long total = (unsigned long long)zero.total_hi << 32 | zero.total_lo;
  const Start st = p.start[w];  // asked for together with worker 0's
  if (w >= L::workers(total) || st.tile == 0) return;
  const unsigned long long u0 = L::part_begin(w, total) - (unsigned)st.tile;  // the block's first tile
  const unsigned w0 = L::worker_of(u0, total), n = L::worker_of(u0 + st.tiles - 1, total) - w0 + 1;
  const int row0 = st.block * L::kBlock;
  const int rows = (int)min((long long)st.n * p.group - row0, (long long)L::kBlock);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
  const int share = (int)((w - w0 - 1) * gridDim.y + blockIdx.y), shares = (int)((n - 1) * gridDim.y);
  const int units = (rows + 31) / 32 * 64;
  // The worker in whose part the block begins has it in slot 1, the others in slot 0.
  const auto slot_of = [&](unsigned i) { return i ? (size_t)2 * (w0 + i) : (size_t)2 * w0 + 1; };
  const auto store = [&](int u, f32x4 x, float m, float l) {
    const int q = u & 63, row = row0 + 32 * (u >> 6) + (lane & 31), node = row / p.group;
    const Out out = out_of(p, st.q0, row, node);
    *reinterpret_cast<u32x2*>(out.o + 16 * q + 8 * h) = scaled<BF16>(x, nothing(l) ? 0.f : 1.f / l);
    if (q == 0 && h == 0 && out.lse) *out.lse = lse_of(m, l);
  };
  // The sums of U units from u on over the parts k0, k0 + step, ..: first their largest
  // maximum, then the sums, 16 loads asked for together.
  const auto sum_parts = [&]<int U>(int u, unsigned k0, unsigned step, f32x4 (&sum)[U], float& m, float& l) {
    constexpr unsigned kAtOnce = 16 / U;
    const int rb = u >> 6, q = u & 63, in = 32 * rb + (lane & 31);
    const auto ml = [&](unsigned k) {
      return *reinterpret_cast<const f32x2*>(p.part + ml_at<RB>(slot_of(min(k, n - 1)), in));
    };
    m = kNone, l = 0.f;
#pragma unroll
    for (int i = 0; i < U; ++i) sum[i] = f32x4{};
    for (unsigned k = k0; k < n; k += 8 * step) {
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = ml(k + e * step).x;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (k + e * step < n) m = __builtin_fmaxf(m, x[e]);
    }
    for (unsigned k = k0; k < n; k += kAtOnce * step) {
      f32x4 x[kAtOnce][U];
      f32x2 v[kAtOnce];
#pragma unroll
      for (unsigned e = 0; e < kAtOnce; ++e) {
        const unsigned i = min(k + e * step, n - 1);
        v[e] = ml(i);
        const f32x4* const at = reinterpret_cast<const f32x4*>(p.part + part_at<RB>(slot_of(i), rb, q) + 4 * lane);
#pragma unroll
        for (int j = 0; j < U; ++j) x[e][j] = at[64 * j];
      }
#pragma unroll
      for (unsigned e = 0; e < kAtOnce; ++e) {
        if (k + e * step >= n) break;
        const float f = __builtin_amdgcn_exp2f(v[e].x - m);
        l += f * v[e].y;
#pragma unroll
        for (int j = 0; j < U; ++j) sum[j] += f * x[e][j];
      }
    }
  };
  if (n <= kFewParts) {
    const auto run = [&]<int U>() {
      for (int u = (share * kJoinWaves + wave) * U; u < units; u += shares * kJoinWaves * U) {
        f32x4 sum[U];
        float m, l;
        sum_parts.template operator()<U>(u, 0, 1, sum, m, l);
        if (32 * (u >> 6) + (lane & 31) < rows)
#pragma unroll
          for (int i = 0; i < U; ++i) store(u + i, sum[i], m, l);
      }
    };
    if (n <= 4)
      run.template operator()<8>();
    else
      run.template operator()<4>();
    return;
  }
  const auto run = [&]<int U>() {
    constexpr int kWords = 4 * U + 2;
    for (int u = share * U; u < units; u += shares * U) {
      f32x4 sum[U];
      float m, l;
      sum_parts.template operator()<U>(u, wave, kJoinWaves, sum, m, l);
      float* const mine = lds + wave * 64 * kWords + lane;  // words 64 apart: a bank a lane
#pragma unroll
      for (int i = 0; i < U; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) mine[64 * (4 * i + e)] = sum[i][e];
      mine[64 * 4 * U] = m, mine[64 * (4 * U + 1)] = l;
      __syncthreads();
      if (wave < U && 32 * (u >> 6) + (lane & 31) < rows) {
        const auto of = [&](int i, int word) { return lds[(i * kWords + word) * 64 + lane]; };
        float m_all = kNone, l_all = 0.f;
#pragma unroll
        for (int i = 0; i < kJoinWaves; ++i) m_all = __builtin_fmaxf(m_all, of(i, 4 * U));
        f32x4 x = {};
#pragma unroll
        for (int i = 0; i < kJoinWaves; ++i) {
          const float f = __builtin_amdgcn_exp2f(of(i, 4 * U) - m_all);
          l_all += f * of(i, 4 * U + 1);
          x += f * f32x4{of(i, 4 * wave), of(i, 4 * wave + 1), of(i, 4 * wave + 2), of(i, 4 * wave + 3)};
        }
        store(u + wave, x, m_all, l_all);
      }
      __syncthreads();
    }
  };
  if (units <= shares)
    run.template operator()<1>();
  else
    run.template operator()<kJoinUnits>();
}

template <bool BF16, int RB>
G9_DEV void fwd(const Params& p, char* smem) {
  using L = Steps<RB>;
  using R = Rows<BF16, RB>;
  constexpr int kAhead = RB - 1;  // steps asked for ahead: the stages of a group but one
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
    // The pages of 32 steps' tiles, two 16-row pieces each, are held in the lanes: a load in
    // every step would be waited for in it, as scalar loads are behind the next LDS read.
    const int* const table = p.table + cur.b * p.table_stride;
    int held;
    const auto hold = [&](int step) {
      const int lane = lane_here(), k = first + (step + (lane >> 1)) * L::kKeys + 16 * (lane & 1);
      held = k < cur.r.keys ? table[k >> p.shift] : -1;
      waitcnt<0, 15>();
    };
    // Piece i of a step's tile of this wave's group.
    const auto piece = [&](int i, int step) {
      return w.aim(i, group * RB + step % RB, first + step * L::kKeys, step < seg ? cur.r.keys : 0,
                   __builtin_amdgcn_readlane(held, 2 * (step & 31) + i));
    };
    const int mine = RB == 4 ? wave >> 1 : wave & 1;
    const auto ask = [&](int step) {
      if constexpr (RB == 1) {
        w.fetch_all(piece(0, step), wave);
        w.fetch_all(piece(1, step), wave);
      } else {
        w.fetch_all(piece(mine, step), wave);
      }
    };
    hold(0);
    ask(0);
    w.load_q(query_of<L>(p, cur, in_block, w.row.node));
    waitcnt<0, 0>();  // here: a wait of the compiler's for the queries would be one in every step
#pragma unroll
    for (int i = 1; i < kAhead; ++i) ask(i);
    w.clear();
    // Rows of this wave, tiles that none of them reads.
    const bool some = cur.block * L::kBlock + 32 * (wave % RB) < cur.r.n * p.group;
    const int whole = min(cur.r.context, cur.r.keys);  // keys that every row reads
    const auto steps = [&]<bool TAIL>(int from, int to) {
#pragma unroll 1
      for (int j = from; j < to; ++j) {
        // The step's tile has landed, for every wave that shares it (a wave of RB 1 has its own).
        waitcnt<(RB == 4 ? 2 * R::kOwn : 0), 15>();
        typename R::Piece next;
        if constexpr (RB > 1) {
          barrier();
          if (((j + kAhead) & 31) == 0) hold(j + kAhead);
          next = piece(mine, j + kAhead);
        } else {
          __builtin_amdgcn_sched_barrier(0);
        }
        const int k0 = first + j * L::kKeys;
        if (some)
          w.template tile<TAIL>(k0, group * RB + j % RB, next, wave);
        else if constexpr (RB > 1)
          w.fetch_all(next, wave);
        if constexpr (RB == 1) {
          waitcnt<63, 0>();
          __builtin_amdgcn_sched_barrier(0);
          if (((j + 1) & 31) == 0) hold(j + 1);
          if (j + 1 < seg) ask(j + 1);
        }
      }
    };
    // The steps whose tiles every row reads whole, then the others.
    const int mid = min(max((whole - cur.tile * L::kKeys) / L::kKeys, 0), seg);
    steps.template operator()<false>(0, mid);
    steps.template operator()<true>(mid, seg);
    settle(w.o);
    const int slot = last && from_start ? -1 : (int)(2 * worker + (from_start ? 1 : 0));
    finish_block<BF16, RB, L>(p, cur, slot, smem, wave, w);
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
  extern "C" __global__ __launch_bounds__(64 * latent::kJoinWaves) void g9_latent_join_##NAME(latent::Params p) { \
    __shared__ float lds[latent::kJoinLds];                                                            \
    latent::join_parts<BF16, RB>(p, lds);                                                                         \
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
  return launched(hipLaunchKernel(kJoin[form][bf16], dim3(fa::kWgs - 1, 2),
                                  dim3(64 * latent::kJoinWaves), args, 0, st));
}
