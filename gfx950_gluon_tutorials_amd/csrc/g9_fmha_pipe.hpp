// The flash-attention pipeline that g9_fmha.hip (equal lengths, whole rows of
// keys) and g9_varlen.hip (packed sequences, causal) run: one workgroup's
// software-pipelined walk over the key tiles.  The layout of its MFMAs and the
// reasons for it are described in g9_fmha.hip.
#pragma once

#include <stdint.h>

#include "g9_common.hpp"

namespace g9 {
namespace fa {

constexpr int kBlockM = 256;                // query rows per workgroup
constexpr int kWaves = 8;
constexpr int kThreads = 64 * kWaves;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kLazyThreshold = 8.f;       // log2 units: p < 256 between rescales

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

// MFMA 32x32x16 on 16-bit operands given as raw registers.
template <bool BF16>
G9_DEV f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                   0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                  0, 0);
}

// Two fp32 values -> one register of two 16-bit values (round to nearest even).
template <bool BF16>
G9_DEV u32 pack2(float x, float y) {
  if constexpr (BF16) {
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(u32, __builtin_convertvector((f32x2){x, y}, b2));
  } else {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(u32, __builtin_convertvector((f32x2){x, y}, h2));
  }
}

// Two 16-bit values of one register -> fp32.
template <bool BF16>
G9_DEV f32x2 unpack2(u32 w) {
  if constexpr (BF16) {
    return f32x2{__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)};
  } else {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    return __builtin_convertvector(__builtin_bit_cast(h2, w), f32x2);
  }
}

// Value of lane l ^ 32 combined with this lane's by a symmetric op.
template <class F>
G9_DEV float xhalf(float x, F op) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_int(x), __float_as_int(x), false, false);
  return op(__int_as_float(r[0]), __int_as_float(r[1]));
}

// Bytes from the first of `rows` rows to the end of the last one, `ld` apart and
// `row` long: a descriptor's range.  Not rows * ld, which leaves out values where
// rows are closer than they are long (expanded or overlapping tensors).
G9_DEV u32 extent(int rows, u32 ld, u32 row) { return rows > 0 ? (u32)(rows - 1) * ld + row : 0; }

// LDS-DMA of 16 bytes per lane (lane i writes lds + 16 i, reading global
// voff + soff) issued as inline assembly, so the compiler does not track it:
// it adds no wait for these DMAs before LDS reads (it cannot tell the read
// addresses from the DMA targets apart and would wait for every DMA in
// flight).  The caller orders them with explicit vmcnt waits and barriers.
// The LDS address goes in through an M0 operand, so the compiler writes M0
// itself and knows what it holds.
G9_DEV void dma16_untracked(rsrc_t r, u32 lds, u32 voff, u32 soff) {
  asm volatile("buffer_load_dwordx4 %1, %2, %3 offen lds" : : "{m0}"(lds), "v"(voff), "s"(r), "s"(soff) : "memory");
}

// The same with a descriptor or offset that the vector unit may just have
// written (v_readfirstlane, or v_readlane where the compiler keeps scalar
// registers in vector lanes): a vector-memory instruction may read such a
// register five wait states later at the earliest, and the compiler, which sees
// to that for its own instructions, does not look into assembly.
G9_DEV void dma16_fresh(rsrc_t r, u32 lds, u32 voff, u32 soff) {
  asm volatile("s_nop 4\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" : : "{m0}"(lds), "v"(voff), "s"(r), "s"(soff) : "memory");
}

// Pins a value to this point of the program: the compiler can neither move
// its computation past the statement nor sink it toward its uses.
G9_DEV void pin(float& x) { asm volatile("" : "+v"(x)); }
G9_DEV void pin(u32& x) { asm volatile("" : "+v"(x)); }
template <class V>
G9_DEV void pin_vec(V& v) {
#pragma unroll
  for (int i = 0; i < (int)(sizeof(V) / 4); ++i) {
    float x = v[i];
    pin(x);
    v[i] = x;
  }
}

G9_DEV u32x2 tr_read(u32 addr) {
  const s16x4 r = __builtin_amdgcn_ds_read_tr16_b64_v4i16((G9_LDS s16x4*)(uintptr_t)addr);
  return __builtin_bit_cast(u32x2, r);
}

// ---------------------------------------------------------------------------
// Pipelined form.  Each wave's loop over key tiles j is cut into four
// clusters, each closed by a workgroup barrier:
//   D1(j)  QK MFMAs of tile j+1 (K_{j+1} from registers) and, in their issue
//          shadow, the second half of tile j's softmax (the remaining
//          exponentials, P_j to 16 bit, the row sum) and, with the eager
//          rescale, half of O's rescale for tile j;
//   M1(j)  LDS reads of V_j; DMA of K_{j+3}; tile j+1's row max, new running
//          max and rescale factor (a dependent chain: it would stall MFMA
//          issue in a dot cluster, here it fills the idle VALU);
//   D2(j)  PV MFMAs of tile j and, in their shadow, most of tile j+1's
//          exponentials;
//   M2(j)  LDS reads of K_{j+2}; DMA of V_{j+2}; rescale of l and (the rest of) O.
// Waves 4-7 run one cluster behind waves 0-3, so on every SIMD one wave is in
// a dot cluster (MFMA + VALU) while the other is in a memory cluster: the
// matrix pipe, the VALU and the LDS / memory pipe are busy at the same time.
// Memory clusters run at wave priority 1, dot clusters at 0, so the memory
// wave's reads, DMAs and rescale win issue arbitration (measured: 2.5% fewer
// loop cycles with the lazy rescale; the priority of M2 is what matters).
// K and V tiles are double buffered in LDS (tile t in buffer t & 1); each DMA
// is waited for (by its own wave, then a barrier) one cluster before the tile
// is read, which gives it about one and a half loop iterations to land.
//
// LDS tiles are stored column-major in 16-byte chunks: chunk c (head-dim
// values 8c..8c+7) of all kBN rows is contiguous (one DMA per 64 rows: lane i
// fetches row i), chunk columns kPitchK / kPitchV bytes apart.  Every LDS read
// address is then one per-lane base register plus an immediate: K reads
// (row = lane % 32 (+32), chunk 2s + lane / 32) cover 256 contiguous bytes per
// 16 lanes; a V transpose read of 16 lanes covers 4 rows of two adjacent
// chunks, 64 bytes each, which the 64-byte pad of kPitchV puts on distinct
// banks.
// ---------------------------------------------------------------------------

#ifndef G9_FMHA_VN1
#define G9_FMHA_VN1 4  // VALU instructions after each QK MFMA of D1
#endif
#ifndef G9_FMHA_VN1_EAGER
#define G9_FMHA_VN1_EAGER 6  // the same with the eager rescale's share of O in D1
#endif
#ifndef G9_FMHA_VN2
#define G9_FMHA_VN2 4  // VALU instructions after each PV MFMA of D2
#endif
#ifndef G9_FMHA_VEC1_EXPS
#define G9_FMHA_VEC1_EXPS 22  // exponentials of a tile done in D2 (of 32 per lane); the rest in D1
#endif

#ifndef G9_FMHA_VN1_SHARED
#define G9_FMHA_VN1_SHARED 3  // VALU instructions after each of D1's 24 QK MFMAs with shared keys
#endif
#ifndef G9_FMHA_VEC1_EXPS_SHARED
#define G9_FMHA_VEC1_EXPS_SHARED 20  // with shared keys: exponentials of a tile (of 32 per lane) done in D2
#endif
#ifndef G9_FMHA_RD1
#define G9_FMHA_RD1 8  // the MFMA of D1 beside which the shared keys' reads begin
#endif

#ifndef G9_FMHA_VN1_64
#define G9_FMHA_VN1_64 8  // head dim 64 (128-key tiles): VALU after each QK MFMA of D1
#endif
#ifndef G9_FMHA_VN2_64
#define G9_FMHA_VN2_64 8  // head dim 64: VALU after each PV MFMA of D2
#endif
#ifndef G9_FMHA_VEC1_EXPS_64
#define G9_FMHA_VEC1_EXPS_64 44  // head dim 64: exponentials of a tile (of 64 per lane) done in D2
#endif

// Sum of a 16-entry table (compile time).
constexpr int sum16(const int (&a)[16]) {
  int t = 0;
  for (int i = 0; i < 16; ++i) t += a[i];
  return t;
}

// SOQ: the scale is folded into Q, so the scores already are in log2 units
// and the exponent argument is a 2-source subtract instead of a 3-source fma
// (fewer register-file reads beside the other wave's LDS returns).
//
// Key tiles are kBN = 8192 / HD keys: 64 at head dim 128, 128 at head dim 64,
// so a dot cluster holds 16 MFMAs either way and the two head dims share the
// per-cluster costs (barriers, the row-max chain, waits) over the same MFMA
// work.  A tile's scores are kNB blocks of 32 keys (Sc).
//
// KIND says where the keys are and which of them a query reads:
//   kEqual   all of p.S rows.
//   kPacked  `keys` rows of one packed sequence, of which each query reads the
//            first `lim` (its causal limit).  Tiles that reach past the wave's
//            smallest limit (`wlim`) are masked by comparing key indexes with
//            lim.  Tile addresses are 64-bit: a descriptor per tile whose range
//            ends with the sequence, so rows behind it read as zeros.
//   kPaged   the tiles from t0 on of a paged request, up to `keys` rows.  A DMA
//            covers eight 16-byte chunks of 8 rows, whole 128-byte lines, which never
//            cross a page.  In
//            LDS, rows go by 8 and chunks of 128 bytes; the groups of K are a
//            chunk further apart and V's rows permuted within a chunk, so that
//            K's reads of 16 rows and V's transposing reads of four chunks touch
//            every bank once.  Which keys from `wlim` on
//            (the request's nodes) a query reads is p's to say (p.reads).  Four
//            tiles of K and of V are in LDS instead of two: the tiles come from
//            HBM, not from an L2 that other workgroups have filled.
enum Kind { kEqual, kPacked, kPaged };
template <class Params, Kind KIND>
struct Where {};
// The request's table row and first tile; the pages of this wave's rows of 64
// tiles, one per lane, and of the next K tile and the next V tile to ask for
// (a scalar load per tile would be waited for in every tile's last cluster:
// 3.3 us a tile instead of 2.4); the query's row in the mask.
template <class Params>
struct Where<Params, kPaged> {
  const int* table;
  int t0, held, pgk, pgv;
  typename Params::Row row;
};
// ROPE: 64 more values of every key, which all heads share: rows of their own,
// behind the key's chunk columns in LDS.  Their fragments are not held: a dot
// cluster D1 reads them beside its first MFMAs, so their buffer is free one cluster
// later than the other columns', and their DMA goes out in M2.
template <int ROPE>
struct SharedKeys {};
template <>
struct SharedKeys<64> {
  const char* rp;  // the sequence's first row
  u32 voffr;       // lane's row offset
};
template <class Params, bool BF16, bool LAZY, bool SOQ, int HD, Kind KIND = kEqual, int ROPE = 0>
struct Pipe : Where<Params, KIND>, SharedKeys<ROPE> {
  static_assert(HD == 64 || HD == 128, "head dim 64 or 128");
  static_assert(ROPE == 0 || (HD == 128 && KIND == kPacked), "shared keys of packed sequences");
  static constexpr int kBN = 8192 / HD;        // keys per tile
  static constexpr int kNB = kBN / 32;         // 32-key score blocks per tile
  static constexpr int kKS = kBN / 16;         // PV steps of 16 keys
  static constexpr int kNS = HD / 16;          // QK steps of 16 head-dim values
  static constexpr int kND = HD / 32;          // PV blocks of 32 head-dim values
  static constexpr int kNC = HD / 8;           // 16-byte chunk columns per row
  static constexpr int kNF = kNS * kNB;        // K (or V) fragments per tile = MFMAs per dot cluster
  static constexpr int kRH = kBN / 64;         // 64-row halves of a chunk column (one DMA each)
  static constexpr int kDW = kNC * kRH / kWaves;  // DMAs per wave per operand and tile
  static constexpr int kPitchK = kBN * 16;     // bytes between K chunk columns
  // Bytes between V chunk columns (pad: distinct banks).
  static constexpr int kPitchV = kBN * 16 + (KIND == kPaged ? 0 : 64);
  static constexpr int kGroupV = kNC * 128, kGroupK = kGroupV + 128;  // kPaged: 8 rows
  static constexpr int kNR = ROPE / 16, kRC = ROPE / 8;  // QK steps and chunk columns of the shared keys
  static constexpr int kTileK = KIND == kPaged ? kBN / 8 * kGroupK : (kNC + kRC) * kPitchK;  // one K tile in LDS
  static constexpr int kTileV = kNC * kPitchV;  // one V tile in LDS
  static constexpr int kBufs = KIND == kPaged ? 4 : 2;  // tiles of K and of V in LDS
  static constexpr int kLdsV = kBufs * kTileK;  // V buffers after the K buffers
  static constexpr int kLdsBytes = kBufs * (kTileK + kTileV);
  static constexpr int kE1 = ROPE ? G9_FMHA_VEC1_EXPS_SHARED : HD == 128 ? G9_FMHA_VEC1_EXPS : G9_FMHA_VEC1_EXPS_64;
  static constexpr int kVN1 = HD == 128 ? G9_FMHA_VN1 : G9_FMHA_VN1_64;
  static constexpr int kVN2 = HD == 128 ? G9_FMHA_VN2 : G9_FMHA_VN2_64;
  static_assert(kNF == 16 && kKS * kND == 16, "16 MFMAs per dot cluster");
  struct Sc {
    f32x16 b[kNB];
  };
  const Params& p;
  int nt, nte, nfull, wave;  // tiles, tiles rounded up to even, whole tiles, wave index
  u32 lds0;
  rsrc_t rk, rv;
  u32 voffk, voffv;  // lane's row offset in global K / V
  u32 ak, av;        // lane's LDS read base for K / V
  float sc;
  u32x4 qf[kNS + kNR];
  u32x4 kv[kNF];  // K_t (kv[kNB s + blk]: step s of 16 head-dim values, key block blk) or V_t (kv[kND t + d])
  f32x16 o[kND];  // O^T, head-dim block d
  float m, l, alpha;
  // Not kEqual: first key's rows (kPaged: of the cache), keys, limits, scratch for P.
  const char *kp, *vp;
  int keys, lim, wlim;
  char* pscratch;
  static constexpr int kScratchBytes = 32 * 32 * 2;  // per wave: P of 32 keys, 16 bit

  G9_DEV explicit Pipe(const Params& pp) : p(pp) {}

  // DMA q = kDW w + i of wave w covers chunk column q / kRH, rows 64 (q % kRH)
  // .. +63 of a tile: lane i fetches row 64 (q % kRH) + i.
  // kPacked: the rows of a tile that the sequence has.  Rows behind them read as
  // zeros, or as values of the last row where rows overlap: masked either way.
  G9_DEV rsrc_t tile_rows(const char* base, int tile, u32 ld, u32 row = HD * 2) const {
    const int left = min(max(keys - tile * kBN, 0), kBN);
    const unsigned long long at = (unsigned long long)base + (unsigned long long)(u32)(tile * kBN) * ld;
    // Uniform, but the 64-bit product may be formed on the vector unit.
    const u32 lo = (u32)__builtin_amdgcn_readfirstlane((int)at), hi = (u32)__builtin_amdgcn_readfirstlane((int)(at >> 32));
    return make_rsrc(reinterpret_cast<const void*>((unsigned long long)hi << 32 | lo),
                     (u32)__builtin_amdgcn_readfirstlane((int)extent(left, ld, row)));
  }
  G9_DEV int first_tile() const {
    if constexpr (KIND == kPaged) return this->t0;
    return 0;
  }
  // The V rows 8 below those at a.
  G9_DEV u32 second(u32 a) const {
    return KIND == kPaged ? a + kGroupV : a + 128;
  }
  // kPaged: lane i's offsets.  A DMA's lane i fetches chunk i / 8 of row i % 8 (V:
  // of row i % 8 ^ 4 (chunk / 2 % 2), see Kind).
  G9_DEV u32 voff_k_of(u32 i) const { return (i & 7) * p.k_t + (i >> 3) * 16; }
  G9_DEV u32 voff_v_of(u32 i) const { return ((i & 7) ^ (i >> 2 & 4)) * p.v_t + (i >> 3) * 16; }
  G9_DEV u32 ak_of(u32 i) const { return lds0 + ((i & 31) >> 3) * kGroupK + (i >> 5) * 128 + (i & 7) * 16; }
  G9_DEV u32 av_of(u32 i) const {
    const u32 G = i >> 4 & 1, jj = i & 15;
    return lds0 + kLdsV + (2 * G + ((jj & 3) >> 1)) * 128 + ((4 * (i >> 5) + (jj >> 2)) ^ (4 * G)) * 16 + 8 * (jj & 1);
  }
  // At head dim 64 they are worked out at each use: held, they and others were
  // spilled, and a reload waits for every DMA in flight (16 x 6000 tokens by 64
  // rows 120 us instead of 66).  At 128 there is room, and neither is better (held
  // and worked out, 64 rows: 4 x 8000 and 200 x 100 tokens 97 and 104, 16 x 6000
  // 101 and 95).
  static constexpr bool kHeld = HD == 128;
  static G9_DEV u32 lane_now() {
    u32 x;
    asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(x));
    return x;
  }
  G9_DEV u32 voff_k() const { return kHeld ? voffk : voff_k_of(lane_now()); }
  G9_DEV u32 voff_v() const { return kHeld ? voffv : voff_v_of(lane_now()); }
  // kPaged: this wave's rows of a tile, 8 by 256 bytes or 16 by 128.
  static constexpr int kMine = kBN / kWaves;
  G9_DEV int my_key(int tile) const { return (this->t0 + tile) * kBN + kMine * wave; }
  G9_DEV void hold_pages(int tile) {
    const int k = my_key(tile + (int)(threadIdx.x & 63));
    this->held = k < keys ? this->table[k >> p.shift] : -1;
    waitcnt<0, 15>();  // here, not at the first use: see dma16_untracked
  }
  G9_DEV int page_of(int tile) const { return __builtin_amdgcn_readlane(this->held, tile & 63); }
  G9_DEV void dma_paged(const char* base, int tile, int page, u32 lds, u32 step_lds, u32 voff, long long step,
                        u32 ld) const {
    const int k = my_key(tile), off = k & ((1 << p.shift) - 1);
    const bool in = (u32)page < (u32)p.num_blocks;
    const int rows = in ? min(max(keys - k, 0), kMine) : 0;
    const unsigned long long at = (unsigned long long)base + (in ? page : 0) * step + (unsigned long long)off * ld;
    const u32 lo = (u32)__builtin_amdgcn_readfirstlane((int)at), hi = (u32)__builtin_amdgcn_readfirstlane((int)(at >> 32));
    const rsrc_t r4 = make_rsrc(reinterpret_cast<const void*>((unsigned long long)hi << 32 | lo),
                                (u32)__builtin_amdgcn_readfirstlane((int)((u32)rows * ld)));
#pragma unroll
    for (int i = 0; i < kDW; ++i) dma16_fresh(r4, lds + i * step_lds, voff, HD == 128 ? i * 128 : i * 8 * ld);
  }
  G9_DEV void dma_k(int tile, int buf) {
    if constexpr (KIND == kPaged) {
      dma_paged(kp, tile, this->pgk, lds0 + buf * kTileK + kMine / 8 * wave * kGroupK, HD == 128 ? 1024 : kGroupK, voff_k(),
                p.k_b, p.k_t);
    } else if constexpr (KIND == kPacked) {
      const rsrc_t r4 = tile_rows(kp, tile, p.ldk);
#pragma unroll
      for (int i = 0; i < kDW; ++i) {
        const int q = kDW * wave + i, c = q / kRH, r = q % kRH;
        dma16_fresh(r4, lds0 + buf * kTileK + c * kPitchK + r * 1024, voffk, 64 * r * p.ldk + c * 16);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kDW; ++i) {
        const int q = kDW * wave + i, c = q / kRH, r = q % kRH;
        dma16_untracked(rk, lds0 + buf * kTileK + c * kPitchK + r * 1024, voffk,
                        ((u32)tile * kBN + 64 * r) * p.ldk + c * 16);
      }
    }
  }
  // The shared keys' chunk column that this wave fetches.
  G9_DEV void dma_r(int tile, int buf) {
    if constexpr (ROPE != 0) {
      static_assert(kRC == kWaves && kRH == 1);
      dma16_fresh(tile_rows(this->rp, tile, p.ldr, ROPE * 2), lds0 + buf * kTileK + (kNC + wave) * kPitchK, this->voffr,
                  wave * 16);
    }
  }
  G9_DEV void dma_v(int tile, int buf) {
    if constexpr (KIND == kPaged) {
      dma_paged(vp, tile, this->pgv, lds0 + kLdsV + buf * kTileV + kMine / 8 * wave * kGroupV, 1024, voff_v(), p.v_b, p.v_t);
    } else if constexpr (KIND == kPacked) {
      const rsrc_t r4 = tile_rows(vp, tile, p.ldv);
#pragma unroll
      for (int i = 0; i < kDW; ++i) {
        const int q = kDW * wave + i, c = q / kRH, r = q % kRH;
        dma16_fresh(r4, lds0 + kLdsV + buf * kTileV + c * kPitchV + r * 1024, voffv, 64 * r * p.ldv + c * 16);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kDW; ++i) {
        const int q = kDW * wave + i, c = q / kRH, r = q % kRH;
        dma16_untracked(rv, lds0 + kLdsV + buf * kTileV + c * kPitchV + r * 1024, voffv,
                        ((u32)tile * kBN + 64 * r) * p.ldv + c * 16);
      }
    }
  }
  // BUF < 0: buffer `buf` (kPaged).
  template <int BUF>
  G9_DEV void read_k(int buf = 0) {
    u32 ak_buf = ak;
    if constexpr (KIND == kPaged) ak_buf = (kHeld ? ak : ak_of(lane_now())) + buf * kTileK;
#pragma unroll
    for (int s = 0; s < kNS; ++s)
#pragma unroll
      for (int blk = 0; blk < kNB; ++blk)
        kv[kNB * s + blk] = *(const G9_LDS u32x4*)(uintptr_t)(
            KIND == kPaged ? ak_buf + 256 * s + 4 * blk * kGroupK : ak + BUF * kTileK + 2 * s * kPitchK + blk * 512);
  }
  template <int BUF>
  G9_DEV void read_v(int buf = 0) {
    u32 av_buf = av;
    if constexpr (KIND == kPaged) av_buf = (kHeld ? av : av_of(lane_now())) + buf * kTileV;
#pragma unroll
    for (int t = 0; t < kKS; ++t)
#pragma unroll
      for (int d = 0; d < kND; ++d) {
        const u32 a = KIND == kPaged ? av_buf + 512 * d + 2 * t * kGroupV : av + BUF * kTileV + 4 * d * kPitchV + 256 * t;
        const u32x2 lo = tr_read(a);
        const u32x2 hi = tr_read(second(a));
        kv[kND * t + d] = u32x4{lo.x, lo.y, hi.x, hi.y};
      }
  }
  // S^T of the tile in kv: kNB 32-key blocks; BUF: where its shared keys are.
  template <int BUF = 0>
  G9_DEV void qk(Sc& S) {
#pragma unroll
    for (int blk = 0; blk < kNB; ++blk) S.b[blk] = mfma<BF16>(kv[blk], qf[0], f32x16{});
#pragma unroll
    for (int s = 1; s < kNS; ++s)
#pragma unroll
      for (int blk = 0; blk < kNB; ++blk) S.b[blk] = mfma<BF16>(kv[kNB * s + blk], qf[s], S.b[blk]);
#pragma unroll
    for (int s = kNS; s < kNS + kNR; ++s)
#pragma unroll
      for (int blk = 0; blk < kNB; ++blk) {
        const u32x4 kr = *(const G9_LDS u32x4*)(uintptr_t)(ak + BUF * kTileK + 2 * s * kPitchK + blk * 512);
        S.b[blk] = mfma<BF16>(kr, qf[s], S.b[blk]);
      }
  }
  // O^T += V^T P^T; P in 16 bit as vec2 left it in S.
  G9_DEV void pv(const Sc& S) {
#pragma unroll
    for (int t = 0; t < kKS; ++t) {
      const f32x16& sv = S.b[t / 2];
      const u32x4 pt = t & 1 ? __builtin_bit_cast(u32x4, __builtin_shufflevector(sv, sv, 8, 9, 10, 11))
                             : __builtin_bit_cast(u32x4, __builtin_shufflevector(sv, sv, 0, 1, 2, 3));
#pragma unroll
      for (int d = 0; d < kND; ++d) o[d] = mfma<BF16>(kv[kND * t + d], pt, o[d]);
    }
  }
  // p = 2^(x * sc - m) for score register i (0 .. 16 kNB - 1) of a lane:
  // block i / 16, register i % 16.
  G9_DEV void expo(Sc& S, int i) const {
    f32x16& v = S.b[i / 16];
    v[i % 16] = __builtin_amdgcn_exp2f(SOQ ? v[i % 16] - m : __builtin_fmaf(v[i % 16], sc, -m));
  }
  // Keys past the sequence end (the phantom tile, or the second half of a
  // 128-key tile when S is an odd multiple of 64) score -inf: their K rows
  // were read as zeros.  `valid` = keys of the tile before the end (a
  // multiple of 64, <= 0 for the phantom).
  G9_DEV void mask(Sc& S, int valid) const {
    const int from = kBN == 64 || valid <= 0 ? 0 : kNB / 2;  // whole-tile stores, no selects
#pragma unroll
    for (int blk = 0; blk < kNB; ++blk)
      if (blk >= from) S.b[blk] = f32x16{} - __builtin_inff();
  }

  // Masked tiles: key 32 blk + 8 (i / 4) + 4 h + i % 4 of the tile scores -inf
  // unless the query reads it.
  G9_DEV void mask_tile(Sc& S, int tile) const {
    const int h = (int)((threadIdx.x & 63) >> 5);
    if constexpr (KIND == kPacked) {
      const int rel = lim - tile * kBN - 4 * h;
#pragma unroll
      for (int blk = 0; blk < kNB; ++blk)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float x = S.b[blk][i];
          S.b[blk][i] = 32 * blk + 8 * (i / 4) + i % 4 < rel ? x : -__builtin_inff();
        }
    } else {
#pragma unroll
      for (int half = 0; half < kRH; ++half) {
        const unsigned long long w = p.reads(this->row, (this->t0 + tile) * kBN + 64 * half, keys);
#pragma unroll
        for (int blk = 2 * half; blk < 2 * half + 2; ++blk) {
          const u32 bits = (u32)(w >> (32 * (blk & 1))) >> (4 * h);
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float x = S.b[blk][i];
            S.b[blk][i] = bits >> (8 * (i / 4) + i % 4) & 1 ? x : -__builtin_inff();
          }
        }
      }
    }
  }
  G9_DEV bool masked(int tile) const { return (first_tile() + tile + 1) * kBN > wlim; }
  // Masked tiles: a weight of 0 does not keep an infinite or NaN value out
  // of the product.  Such values (rare: one packed maximum over V's registers
  // finds them) are taken out of the registers, and added on the vector unit to
  // the rows that may read their key.  V_tile is in buffer `buf` and in kv, P_tile
  // in S as vec2 left it.
  G9_DEV void guard_v(const Sc& S, int tile, int buf) {
    typedef unsigned short h2 __attribute__((ext_vector_type(2)));
    constexpr u32 kExp = BF16 ? 0x7f80u : 0x7c00u;
    h2 top = {0, 0};
#pragma unroll
    for (int f = 0; f < kNF; ++f)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        top = __builtin_elementwise_max(top, __builtin_bit_cast(h2, kv[f][e] & 0x7fff7fffu));
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(top.x >= kExp || top.y >= kExp) == 0, 1)) return;
#pragma unroll
    for (int f = 0; f < kNF; ++f)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        u32 x = kv[f][e];
        if ((x & kExp) == kExp) x &= 0xffff0000u;
        if (((x >> 16) & kExp) == kExp) x &= 0xffffu;
        pin(x);  // one compare at a time: their masks would not fit the scalar registers
        kv[f][e] = x;
      }
    // 32 keys at a time: P in LDS, row of the query, column of the key.
    const int lane = threadIdx.x & 63, h = lane >> 5;
    uint16_t* const prow = reinterpret_cast<uint16_t*>(pscratch) + (lane & 31) * 32;
    const int first = (first_tile() + tile) * kBN;
#pragma unroll
    for (int blk = 0; blk < kNB; ++blk) {
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        const u32 w = __float_as_uint(S.b[blk][8 * (i / 8) + (i % 8) / 2]);
        *reinterpret_cast<u32*>(prow + 8 * (i / 4) + 4 * h + i % 4) = w;
      }
      waitcnt<63, 0>();
      const int from = first + 32 * blk;
      unsigned long long who = 0;
      if constexpr (KIND == kPaged)
        who = p.reads(this->row, from, keys);
      else
        who = lim - from >= 64 ? ~0ull : lim - from <= 0 ? 0 : (1ull << (lim - from)) - 1;
#pragma unroll 1
      for (int key = 0; key < 32; ++key) {
        if (!((who >> key) & 1)) continue;
        const float w = unpack2<BF16>(prow[key]).x;
        const int kt = 32 * blk + key;
        const u32 a = lds0 + kLdsV + buf * kTileV + 8 * h + (KIND == kPaged ? (kt >> 3) * kGroupV : kt * 16);
#pragma unroll
        for (int d = 0; d < kND; ++d)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const u32x2 x = *(const G9_LDS u32x2*)(uintptr_t)(
                a + (KIND == kPaged ? (4 * d + r) * 128 + ((key & 7) ^ (4 * (r >> 1))) * 16 : (4 * d + r) * kPitchV));
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
  }

  // Start of a tile's softmax: row max, running max and alpha (a dependent
  // chain ending in a cross-lane exchange; run in a memory cluster, where the
  // VALU is otherwise idle, so the MFMA shadows keep only independent work).
  // One max3 chain per 8-register half block, then a tree over the chains.
  G9_DEV void vec0(Sc& S) {
    float c[2 * kNB];
#pragma unroll
    for (int h = 0; h < 2 * kNB; ++h) {
      const f32x16& v = S.b[h / 2];
      const int o8 = 8 * (h & 1);
      c[h] = __builtin_fmaxf(__builtin_fmaxf(v[o8], v[o8 + 1]), v[o8 + 2]);
    }
#pragma unroll
    for (int i = 3; i < 8; i += 2) {
      const int i1 = i + 1 < 8 ? i + 1 : i;
#pragma unroll
      for (int h = 0; h < 2 * kNB; ++h) {
        const f32x16& v = S.b[h / 2];
        const int o8 = 8 * (h & 1);
        c[h] = __builtin_fmaxf(__builtin_fmaxf(c[h], v[o8 + i]), v[o8 + i1]);
      }
    }
#pragma unroll
    for (int w = 2 * kNB; w > 1; w /= 2)
#pragma unroll
      for (int h = 0; h < w / 2; ++h) c[h] = __builtin_fmaxf(c[2 * h], c[2 * h + 1]);
    float mx = c[0];
    mx = xhalf(mx, [](float x, float y) { return __builtin_fmaxf(x, y); });
    const float mt = SOQ ? mx : mx * sc;
    const float m_new = LAZY ? (mt - m > kLazyThreshold ? mt : m) : __builtin_fmaxf(m, mt);
    alpha = __builtin_amdgcn_exp2f(m - m_new);
    m = m_new;
  }
  // First kE1 exponentials of a tile (in place).
  G9_DEV void vec1(Sc& S) {
#pragma unroll
    for (int i = 0; i < kE1; ++i) expo(S, i);
  }
  // Second half: the remaining exponentials, l += row sum (fp32, before
  // rounding), P to 16 bit.  The 16-bit pairs of PV step t are written over
  // the first four registers of their eight scores (registers 8(t % 2) .. +3
  // of block t / 2), so P needs no registers of its own.  (The row sum uses
  // plain adds: v_dot2c on the packed values would take half the
  // instructions but does not issue beside an MFMA -- measured: two per MFMA
  // stretch its 32-cycle interval to 53.)
  G9_DEV void vec2(Sc& S) {
#pragma unroll
    for (int i = kE1; i < 16 * kNB; ++i) expo(S, i);
    float r[2 * kNB];
#pragma unroll
    for (int h = 0; h < 2 * kNB; ++h) {
      const f32x16& v = S.b[h / 2];
      const int o8 = 8 * (h & 1);
      r[h] = v[o8] + v[o8 + 1];
    }
#pragma unroll
    for (int i = 2; i < 8; ++i)
#pragma unroll
      for (int h = 0; h < 2 * kNB; ++h) r[h] += S.b[h / 2][8 * (h & 1) + i];
#pragma unroll
    for (int w = 2 * kNB; w > 1; w /= 2)
#pragma unroll
      for (int h = 0; h < w / 2; ++h) r[h] = r[2 * h] + r[2 * h + 1];
    l += r[0];
#pragma unroll
    for (int t = 0; t < kKS; ++t) {
      f32x16& sv = S.b[t / 2];
      const int r0 = 8 * (t & 1);
#pragma unroll
      for (int e = 0; e < 4; ++e) sv[r0 + e] = __uint_as_float(pack2<BF16>(sv[r0 + 2 * e], sv[r0 + 2 * e + 1]));
    }
  }
  // Pins the 16-bit P pairs and l (vec2's results).
  G9_DEV void pin_p(Sc& S) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int blk = 0; blk < kNB; ++blk) {
        float a = S.b[blk][e], b = S.b[blk][8 + e];
        pin(a), pin(b);
        S.b[blk][e] = a, S.b[blk][8 + e] = b;
      }
    pin(l);
  }
  G9_DEV void pin_sc(Sc& S) {
#pragma unroll
    for (int blk = 0; blk < kNB; ++blk) pin_vec(S.b[blk]);
  }
  // The eager rescale (every tile) at head dim 128 splits O: the first kSplit
  // head-dim blocks are rescaled in the next dot cluster, as VALU work beside
  // the QK MFMAs (rescale_early), the rest here (measured: 7.5% fewer loop
  // cycles than all of it here; at head dim 64, whose dot clusters have half
  // the MFMAs, 1.5% more).  The lazy rescale is rare and stays here whole.
  // Both skip the multiplies here when no row of the wave moved its max
  // (alpha is then exactly 1, so the skip changes no bit; eager rescale: 1.8%
  // fewer loop cycles at S=8192, where later tiles rarely move a row's max).
  static constexpr int kSplit = LAZY || HD != 128 ? 0 : kND / 2;
  G9_DEV void rescale() {
    l *= alpha;
    if (__builtin_amdgcn_ballot_w64(alpha != 1.f)) {
#pragma unroll
      for (int d = kSplit; d < kND; ++d) o[d] *= alpha;
    }
  }
  G9_DEV void rescale_early() {
#pragma unroll
    for (int d = 0; d < kSplit; ++d) o[d] *= alpha;
  }

  // Interleave of a dot cluster (kNF MFMAs): MFMA i followed by VN VALU
  // instructions and exps_in_slot() exponentials.  An MFMA 32x32x16 takes 32
  // cycles; about six plain VALU instructions or two to three exponentials
  // issue beside it without delaying the next one (measured).  Exponentials
  // are not in the VALU class of sched_group_barrier; left to the scheduler
  // they bunch up (5-8 in one MFMA slot, none in the next ten), so each slot
  // gets its own count.  D1 (W = 1) finishes tile j's exponentials, which its
  // row sums and 16-bit conversions consume later in the same cluster, so
  // they go early; D2 (W = 2) starts tile j+1's, which nothing in D2 reads,
  // so they are spread out.  The counts were chosen by measurement (loop
  // cycles at B=32 S=8192 bf16: head dim 128 v4 -3.4%, v3 +-0; head dim 64
  // -3.8% and -3.0% against the spread the scheduler picks; the sum over a
  // cluster is the exponentials it holds: 10 and 22 of 32 at head dim 128,
  // 20 and 44 of 64 at 64).
  static constexpr int kEp1[16] = {1, 1, 1, 1, 1, 1, 1, 1, 1, 1};  // D1, lazy rescale
  static constexpr int kEp1e[16] = {4, 3, 3};  // D1 beside the eager rescale's 6 VALU per slot
  static constexpr int kEp2[16] = {1, 1, 2, 2, 2, 2, 2, 2, 2, 2, 2, 2};
  static constexpr int kEp1_64[16] = {1, 1, 1, 1, 2, 2, 2, 2, 2, 2, 2, 2};
  static constexpr int kEp2_64[16] = {2, 3, 3, 3, 3, 3, 3, 3, 3, 3, 3, 3, 3, 3, 3};
  // With shared keys: `all` exponentials over the first `slots` slots.
  static constexpr int shared_exps(int i, int all, int slots) {
    return i < slots ? (i + 1) * all / slots - i * all / slots : 0;
  }
  template <int W, int I>
  G9_DEV static constexpr int exps_in_slot() {
    if constexpr (ROPE != 0)
      return W == 1 ? shared_exps(I, 32 - kE1, kNF) : shared_exps(I, kE1, kNF - 2);
    else if constexpr (HD == 128)
      return W == 1 ? (LAZY ? kEp1[I] : kEp1e[I]) : kEp2[I];
    else
      return W == 1 ? kEp1_64[I] : kEp2_64[I];
  }
  static_assert(HD != 128 || ROPE || sum16(kEp1) == 32 - kE1, "D1 exponentials per slot: re-chosen with the D1/D2 split");
  static_assert(HD != 128 || ROPE || sum16(kEp1e) == 32 - kE1, "D1 exponentials per slot: re-chosen with the D1/D2 split");
  static_assert(HD != 128 || ROPE || sum16(kEp2) == kE1, "D2 exponentials per slot: re-chosen with the D1/D2 split");
  static_assert(HD == 128 || sum16(kEp1_64) == 64 - kE1, "D1 exponentials per slot: re-chosen with the D1/D2 split");
  static_assert(HD == 128 || sum16(kEp2_64) == kE1, "D2 exponentials per slot: re-chosen with the D1/D2 split");
  template <int VN, int W, int I = 0>
  G9_DEV static void interleave() {
    if constexpr (I < kNF) {
      __builtin_amdgcn_sched_group_barrier(SG_MFMA, 1, 0);
      __builtin_amdgcn_sched_group_barrier(SG_VALU, VN, 0);
      constexpr int e = exps_in_slot<W, I>();
      if constexpr (e > 0) __builtin_amdgcn_sched_group_barrier(SG_TRANS, e, 0);
      interleave<VN, W, I + 1>();
    }
  }

  // D1 with the shared keys: 24 MFMAs; eight LDS reads go beside the 9th to the 16th, whose
  // registers they take.
  template <int VN, int I = 0>
  G9_DEV static void interleave_shared() {
    if constexpr (I < kNF + kNR * kNB) {
      __builtin_amdgcn_sched_group_barrier(SG_MFMA, 1, 0);
      if constexpr (I >= G9_FMHA_RD1 && I < G9_FMHA_RD1 + kNR * kNB) __builtin_amdgcn_sched_group_barrier(SG_DS_RD, 1, 0);
      __builtin_amdgcn_sched_group_barrier(SG_VALU, VN, 0);
      constexpr int e = exps_in_slot<1, I>();
      if constexpr (e > 0) __builtin_amdgcn_sched_group_barrier(SG_TRANS, e, 0);
      interleave_shared<VN, I + 1>();
    }
  }

  // Not kEqual: V_{j+1} landed, for a wave that has no more use for it.
  G9_DEV void wait_v(int j) const {
    if (j + 1 >= nte) return;
    if (KIND == kPaged ? j + 5 < nte : j + 3 < nte)
      waitcnt<(KIND == kPaged ? 5 : 1) * kDW, 15>();
    else
      waitcnt<0, 15>();
  }
  // kPaged: M2(j)'s DMA, and the pages of the next ones.
  G9_DEV void ask_v(int j) {
    if (j + 4 < nte) dma_v(j + 4, j & 3);
    this->pgv = this->pgk;  // tile j + 5's V is asked for next, tile j + 6's K
    if (((j + 6) & 63) == 0) hold_pages(j + 6);
    this->pgk = page_of(j + 6);
  }
  // Not kEqual: iteration j of a wave none of whose rows reads tile j or one
  // behind it: its share of the DMAs and the barriers.
  G9_DEV void idle(int j) {
    barrier();
    if constexpr (KIND == kPaged) {
      if (j + 4 < nte)
        waitcnt<5 * kDW, 15>();
      else
        waitcnt<0, 15>();
      if (j + 5 < nte) dma_k(j + 5, (j + 1) & 3);
    } else {
      if (j + 2 < nte) waitcnt<kDW, 15>();
      if (j + 3 < nte) dma_k(j + 3, (j & 1) ^ 1);
    }
    barrier();
    barrier();
    wait_v(j);
    if constexpr (KIND == kPaged) {
      ask_v(j);
    } else {
      if constexpr (ROPE != 0)
        if (j + 3 < nte) dma_r(j + 3, (j & 1) ^ 1);
      if (j + 2 < nte) dma_v(j + 2, j & 1);
    }
    barrier();
  }

  // One loop iteration; PAR = j & 1 fixes the LDS buffers; c holds tile j's
  // scores after vec1, n receives tile j+1's; NEXT: tile j+1 exists.  The
  // loop runs over an even number of tiles nte: when nt is odd the last tile
  // is a phantom past the end of the sequence (its DMAs read zeros from the
  // buffer range check) whose scores are set to -inf, so it adds nothing.
  // Registers are written unconditionally (a read past the last tile reads a
  // stale but in-bounds buffer), so no value has to survive a skipped branch.
  template <int PAR, bool NEXT>
  G9_DEV void step(int j, Sc& c, Sc& n) {
    // D1(j)
    __builtin_amdgcn_s_setprio(0);
    if constexpr (NEXT) {
      if constexpr (ROPE != 0)
        qk<PAR ^ 1>(n);
      else
        qk(n);
      vec2(c);
      rescale_early();
      if constexpr (ROPE != 0)
        interleave_shared<G9_FMHA_VN1_SHARED>();
      else
        interleave<(kSplit ? G9_FMHA_VN1_EAGER : kVN1), 1>();
      pin_sc(n);
    } else {
      vec2(c);
      rescale_early();
    }
#pragma unroll
    for (int d = 0; d < kSplit; ++d) pin_vec(o[d]);
    pin_p(c);
    barrier();
    // M1(j): V_j was waited for at the end of M2(j-1) (or the prologue).
    __builtin_amdgcn_s_setprio(1);
    if constexpr (KIND == kPaged) {
      read_v<-1>(j & 3);
      if (j + 4 < nte)
        waitcnt<5 * kDW, 15>();  // K_{j+2} landed; V_{j+1}, K_{j+3}, V_{j+2}, K_{j+4}, V_{j+3} may be in flight
      else
        waitcnt<0, 15>();
      if (j + 5 < nte) dma_k(j + 5, (j + 1) & 3);
    } else {
      read_v<PAR>();
      if (j + 2 < nte) waitcnt<kDW, 15>();  // K_{j+2} landed (V_{j+1} may be in flight)
      if (j + 3 < nte) dma_k(j + 3, PAR ^ 1);
    }
    if constexpr (NEXT) {
      if constexpr (KIND != kEqual) {
        if (masked(j + 1)) {
          asm volatile("");
          mask_tile(n, j + 1);
        }
      } else if (j + 1 >= nfull) {  // past the end (a branch, not selects in every step)
        asm volatile("");
        mask(n, p.S - (j + 1) * kBN);
      }
      vec0(n);
      pin(m);
      pin(alpha);
    }
    waitcnt<63, 0>();
    if constexpr (KIND != kEqual)
      if (masked(j)) guard_v(c, j, KIND == kPaged ? j & 3 : PAR);
    barrier();
    // D2(j)
    __builtin_amdgcn_s_setprio(0);
    if constexpr (NEXT) {
      pv(c);
      vec1(n);
      interleave<kVN2, 2>();
      pin_sc(n);
    } else {
      pv(c);
    }
#pragma unroll
    for (int d = 0; d < kND; ++d) pin_vec(o[d]);
    barrier();
    // M2(j)
    __builtin_amdgcn_s_setprio(1);
    if constexpr (NEXT) {
      if constexpr (KIND == kPaged) {
        read_k<-1>((j + 2) & 3);
        if (j + 5 < nte)
          waitcnt<5 * kDW, 15>();  // V_{j+1} landed; K_{j+3}, V_{j+2}, K_{j+4}, V_{j+3}, K_{j+5} may be in flight
        else
          waitcnt<0, 15>();
      } else {
        read_k<PAR>();
        if (j + 3 < nte)
          waitcnt<kDW, 15>();  // V_{j+1} landed (K_{j+3} may be in flight)
        else
          waitcnt<0, 15>();
      }
      rescale();
    }
    // Not kEqual: a wave's last tile need not be the workgroup's.
    if constexpr (KIND != kEqual && !NEXT) wait_v(j);
    if constexpr (KIND == kPaged) {
      ask_v(j);
    } else {
      if constexpr (ROPE != 0)
        if (j + 3 < nte) dma_r(j + 3, PAR ^ 1);
      if (j + 2 < nte) dma_v(j + 2, PAR);
    }
    waitcnt<63, 0>();
    barrier();
  }
};

}  // namespace fa
}  // namespace g9
