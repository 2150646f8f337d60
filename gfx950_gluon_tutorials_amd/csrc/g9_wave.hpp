// One wave's attention over key tiles of its own: 32 (head dim 128) or 64 keys in
// LDS, filled by LDS-DMA in stages of 8 KB of K and 8 KB of V.  The short packed
// kernel (g9_varlen.hip) and the paged one (g9_tree.hip) run it.
//
// Per tile a wave computes S^T = K Q^T and O^T += V^T P^T with 32x32x16 MFMAs in
// the register layouts that g9_fmha.hip describes: the scores are the second
// product's operand as they stand, V is read by transposing LDS reads.  The weights
// P are rounded to the 16-bit type for that product, whose operands are of one type
// (fp32 products have a sixteenth of the rate); their sum l is taken before.
#pragma once

#include "g9_fmha_pipe.hpp"

namespace g9 {
namespace fa {

template <class V>
G9_DEV V uniform(V x) {
  if constexpr (sizeof(V) == 8) {
    const unsigned long long u = (unsigned long long)x;
    const u32 lo = (u32)__builtin_amdgcn_readfirstlane((int)u), hi = (u32)__builtin_amdgcn_readfirstlane((int)(u >> 32));
    return (V)((unsigned long long)hi << 32 | lo);
  } else {
    return (V)__builtin_amdgcn_readfirstlane((int)x);
  }
}

// p.reads says which keys a row reads, p.scale_log2 the scale.
// NQ groups of 32 query rows, which share every K and V register read from LDS.
template <class Params, bool BF16, int HD, int NQ, int STAGES = 2>
struct Wave {
  static constexpr int kKeys = 4096 / HD;          // keys per tile
  static constexpr int kNB = kKeys / 32;           // 32-key score blocks
  static constexpr int kNS = HD / 16;              // QK steps of 16 head-dim values
  static constexpr int kKS = kKeys / 16;           // PV steps of 16 keys
  static constexpr int kND = HD / 32;              // PV blocks of 32 head-dim values
  static constexpr int kRow = HD * 2;              // bytes of a row
  static constexpr int kRows = 1024 / kRow;        // rows of one DMA
  static constexpr int kPieces = kKeys / 16;       // 16-row pieces: never across a page
  static constexpr int kDmas = 8;                  // per tile and operand
  static constexpr int kStage = 16384, kV = 8192;  // a stage; V behind K
  static constexpr int kScratch = 32 * kKeys * 2;  // P of one tile and 32 rows, 16 bit
  static constexpr int kWaveLds = STAGES * kStage + kScratch;

  const Params& p;
  int lane, h, col;  // lane, lane / 32, lane % 32
  u32 lds;           // this wave's LDS
  char* scratch;
  u32 voffk[4], voffv[1];
  u32 ak, av;        // LDS read bases in a stage (K, V)
  u32x4 qf[NQ][kNS];
  f32x16 o[NQ][kND];
  float m[NQ], l[NQ];
  int node[NQ];      // of this lane's queries, -1 where there is none
  int context, q0, keys;  // of the request

  G9_DEV explicit Wave(const Params& pp) : p(pp) {}

  // LDS layout of a tile: rows of kRow bytes, their 16-byte chunks permuted
  // within the row so that a read of one chunk from 16 rows (K), or of 64 bytes
  // from 4 rows (V), touches every bank once.  Chunk c of row r is at slot c ^
  // swz(r).  An LDS-DMA writes lane i's 16 bytes at 16 i, so lane i fetches the
  // chunk that belongs there; a wave's DMA reads whole rows.
  static G9_DEV int swz_k(int r) { return HD == 128 ? r & 15 : (r >> 1) & 7; }
  static G9_DEV int swz_v(int r) { return HD == 128 ? 4 * (r & 3) : 4 * ((r >> 1) & 1); }

  G9_DEV void init(char* smem, int wave, u32 k_t, u32 v_t) {
    lane = threadIdx.x & 63, h = lane >> 5, col = lane & 31;
    lds = (u32)(uintptr_t)to_lds(smem) + wave * kWaveLds;
    scratch = smem + wave * kWaveLds + STAGES * kStage;
    constexpr int kPer = kRow / 16;  // chunks of a row
    const int r = lane / kPer, slot = lane % kPer;
#pragma unroll
    for (int j = 0; j < 4; ++j) voffk[j] = r * k_t + 16 * (slot ^ swz_k(kRows * j + r));
    voffv[0] = r * v_t + 16 * (slot ^ swz_v(r));
    // K: row col, chunk 2 s + h.  V's transposing reads: 16 lanes cover 4 rows and
    // 16 values; lane jj of them addresses row jj / 4 and values 4 (jj % 4) of
    // chunk 4 d + 2 (lane / 16 % 2) + jj / 2 % 2.  Steps and blocks come in by XOR
    // (of whole bit fields: the rows are aligned to their size).
    const int jj = lane & 15, r4 = 4 * h + (jj >> 2);
    ak = lds + col * kRow + 16 * (h ^ swz_k(col));
    av = lds + kV + r4 * kRow + 16 * ((2 * (lane >> 4 & 1) + ((jj & 3) >> 1)) ^ swz_v(r4)) + 8 * (jj & 1);
  }

  // Rows 16 i .. 16 i + 15 of a tile, `rows` of them there (the others read as
  // zeros, or as values of the last one where rows overlap), K's at k, V's at v, k_t
  // and v_t bytes apart.
  G9_DEV void fill_piece(int i, int stage, const char* k, const char* v, int rows, u32 k_t, u32 v_t) const {
    const rsrc_t rk = make_rsrc(uniform(k), uniform(extent(rows, k_t, kRow)));
    const rsrc_t rv = make_rsrc(uniform(v), uniform(extent(rows, v_t, kRow)));
#pragma unroll
    for (int jj = 0; jj < 16 / kRows; ++jj) {
      const int j = i * (16 / kRows) + jj;
      dma16_fresh(rk, lds + stage * kStage + j * 1024, voffk[j & (HD == 128 ? 3 : 1)], jj * kRows * k_t);
      dma16_fresh(rv, lds + stage * kStage + kV + j * 1024, voffv[0], jj * kRows * v_t);
    }
  }
  G9_DEV void load_q(int t, const char* qrow) {
#pragma unroll
    for (int s = 0; s < kNS; ++s) qf[t][s] = *reinterpret_cast<const u32x4*>(qrow + (16 * s + 8 * h) * 2);
  }
  G9_DEV void clear() {
#pragma unroll
    for (int t = 0; t < NQ; ++t) {
      // Finite, so that a row that has read nothing yet has weights 2^(-inf - m) =
      // 0 and a sum of 0, not NaN.
      m[t] = -3.0e38f, l[t] = 0.f;
#pragma unroll
      for (int d = 0; d < kND; ++d) o[t][d] = f32x16{};
    }
  }

  // Adds the tile of the keys from k0 on; tail: not every row reads all of them.
  G9_DEV void tile(int k0, int stage, bool tail) {
    f32x16 sc[NQ][kNB];
    const u32 ak_s = ak + stage * kStage, av_s = av + stage * kStage;
#pragma unroll
    for (int s = 0; s < kNS; ++s)
#pragma unroll
      for (int b = 0; b < kNB; ++b) {
        const u32x4 kf = *(const G9_LDS u32x4*)(uintptr_t)((ak_s ^ (32 * s)) + 32 * b * kRow);
#pragma unroll
        for (int t = 0; t < NQ; ++t) sc[t][b] = mfma<BF16>(kf, qf[t][s], s ? sc[t][b] : f32x16{});
      }
    u32x4 pf[NQ][kKS];
#pragma unroll
    for (int t = 0; t < NQ; ++t) {
      if (tail) {
        const unsigned long long w = p.reads({node[t], context, q0}, k0, keys);
#pragma unroll
        for (int b = 0; b < kNB; ++b) {
          const u32 bits = (u32)(w >> (32 * b)) >> (4 * h);
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float x = sc[t][b][i];
            sc[t][b][i] = bits >> (8 * (i / 4) + i % 4) & 1 ? x : -__builtin_inff();
          }
        }
      }
      float top = sc[t][0][0];
#pragma unroll
      for (int b = 0; b < kNB; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) top = __builtin_fmaxf(top, sc[t][b][i]);
      top = xhalf(top, [](float x, float y) { return __builtin_fmaxf(x, y); });
      const float m_new = __builtin_fmaxf(m[t], top * p.scale_log2);
      const float alpha = __builtin_amdgcn_exp2f(m[t] - m_new);
      m[t] = m_new;
      float sum[4] = {};
#pragma unroll
      for (int b = 0; b < kNB; ++b)
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][b][i], p.scale_log2, -m_new));
          const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][b][i + 1], p.scale_log2, -m_new));
          sum[i / 2 % 2 * 2] += x, sum[i / 2 % 2 * 2 + 1] += y;
          pf[t][2 * b + i / 8][i % 8 / 2] = pack2<BF16>(x, y);
        }
      l[t] = l[t] * alpha + ((sum[0] + sum[1]) + (sum[2] + sum[3]));
      if (__builtin_amdgcn_ballot_w64(alpha != 1.f)) {
#pragma unroll
        for (int d = 0; d < kND; ++d) o[t][d] *= alpha;
      }
    }
    if (tail) guard(k0, stage, pf);
#pragma unroll
    for (int k = 0; k < kKS; ++k)
#pragma unroll
      for (int d = 0; d < kND; ++d) {
        // And the rows 8 below: their chunks are permuted alike.
        const u32 a = (av_s ^ (64 * d)) + 16 * k * kRow;
        const u32x2 lo = tr_read(a), hi = tr_read(a + 8 * kRow);
        const u32x4 vf = {lo.x, lo.y, hi.x, hi.y};
#pragma unroll
        for (int t = 0; t < NQ; ++t) o[t][d] = mfma<BF16>(vf, pf[t][k], o[t][d]);
      }
  }

  // Tails: a weight of 0 does not keep an infinite or NaN value
  // out of the product.  Such values (rare) are added on the vector unit to the
  // rows that read their key, and then taken out of the tile.
  G9_DEV void guard(int k0, int stage, const u32x4 (&pf)[NQ][kKS]) {
    typedef unsigned short h2 __attribute__((ext_vector_type(2)));
    constexpr u32 kExp = BF16 ? 0x7f80u : 0x7c00u;
    G9_LDS u32x4* const mine = (G9_LDS u32x4*)(uintptr_t)(lds + stage * kStage + kV + lane * 16);
    h2 top = {0, 0};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const u32x4 x = mine[64 * j];
#pragma unroll
      for (int e = 0; e < 4; ++e) top = __builtin_elementwise_max(top, __builtin_bit_cast(h2, x[e] & 0x7fff7fffu));
    }
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(top.x >= kExp || top.y >= kExp) == 0, 1)) return;
    // P in LDS, 32 rows at a time: row of the query, column of the key.
    uint16_t* const prow = reinterpret_cast<uint16_t*>(scratch) + col * kKeys;
#pragma unroll
    for (int t = 0; t < NQ; ++t) {
#pragma unroll
      for (int k = 0; k < kKS; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          *reinterpret_cast<u32*>(prow + 16 * k + 8 * (e >> 1) + 4 * h + 2 * (e & 1)) = pf[t][k][e];
      const unsigned long long w = p.reads({node[t], context, q0}, k0, keys);
      waitcnt<63, 0>();
#pragma unroll 1
      for (int key = 0; key < kKeys; ++key) {
        if (!((w >> key) & 1)) continue;
        const float wt = unpack2<BF16>(prow[key]).x;
        const u32 vr = lds + stage * kStage + kV + key * kRow;
#pragma unroll
        for (int d = 0; d < kND; ++d)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const u32x2 x = *(const G9_LDS u32x2*)(uintptr_t)(vr + 16 * ((4 * d + r) ^ swz_v(key)) + 8 * h);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              u32 y = (e & 1 ? x[e / 2] >> 16 : x[e / 2]) & 0xffffu;
              if ((y & kExp) != kExp) y = 0;
              o[t][d][4 * r + e] += wt * unpack2<BF16>(y).x;
            }
            __builtin_amdgcn_sched_barrier(0);
          }
      }
    }
#pragma unroll 1
    for (int j = 0; j < 8; ++j) {
      u32x4 x = mine[64 * j];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if ((x[e] & kExp) == kExp) x[e] &= 0xffff0000u;
        if (((x[e] >> 16) & kExp) == kExp) x[e] &= 0xffffu;
      }
      mine[64 * j] = x;
    }
    waitcnt<63, 0>();
  }
};

}  // namespace fa
}  // namespace g9
