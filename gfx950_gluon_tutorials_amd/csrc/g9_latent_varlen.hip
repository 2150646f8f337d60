// Attention over packed sequences whose keys and values were expanded from
// latents (g9_latent_varlen_fwd, include/gfx950_fmha.h): a head's key is 128 values
// of its own and 64 rotated ones that all heads share, its value 128.
//
// g9_varlen.hip's kernel with 192 values of QK: the pipeline reads the shared keys as
// chunk columns of their own behind the head's, so that nothing is copied together.
// Bound by the matrix unit (640 flops a query and key of a head): 16384 causal tokens by 32
// heads 2.28-2.66 ms on several cards (1.03-1.21 PFLOP/s, where a large matrix product has 1.40-1.52).
// On one of 2.35 ms it is busy for 64% of the cycles, which the power limit holds at 1.77 GHz;
// a tenth of the waves' time is waits for LDS, and 1% of the products are masked.  12 prompts of 100
// to 2500 by 32 heads 336-386 us (0.70-0.80 PFLOP/s): busy for 41% at 1.92 GHz, 8% of the products
// masked; the rest is the beginnings and ends of 1600 workgroups, one a CU at a time.  197
// tokens by 16 heads 8 us in the short form.
#include "../../include/gfx950_fmha.h"
#include "g9_attn_host.hpp"
#include "g9_packed.hpp"

namespace g9 {
namespace fa {

struct LatentVarParams : VarParams {
  const char* r;  // the shared keys, ldr bytes a token
  u32 ldr;
};

}  // namespace fa
}  // namespace g9

using namespace g9;
using namespace g9::host;

#define G9_LATENT_VARLEN_KERNEL(NAME, BF16)                                                                   \
  extern "C" __global__ __launch_bounds__(fa::kThreads) __attribute__((amdgpu_waves_per_eu(2, 2))) void      \
  NAME(fa::LatentVarParams p) {                                                                              \
    __shared__ __attribute__((aligned(1024))) char smem[fa::VarPipe<fa::LatentVarParams, BF16, 128, 64>::kLds]; \
    fa::varlen_fwd<BF16, 128, 64>(p, smem);                                                                  \
  }
#define G9_LATENT_SHORT_KERNEL(NAME, BF16)                                                                    \
  extern "C" __global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) void               \
  NAME(fa::LatentVarParams p) {                                                                              \
    __shared__ __attribute__((aligned(1024))) char smem[fa::ShortWave<fa::LatentVarParams, BF16, 128, 64>::kLds]; \
    fa::varlen_short<BF16, 128, 64>(p, smem);                                                                \
  }
G9_LATENT_SHORT_KERNEL(g9_latent_varlen_short_bf16, true)
G9_LATENT_SHORT_KERNEL(g9_latent_varlen_short_f16, false)
G9_LATENT_VARLEN_KERNEL(g9_latent_varlen_bf16, true)
G9_LATENT_VARLEN_KERNEL(g9_latent_varlen_f16, false)

// The short form runs up to this many rows (queries by query heads), and where the sequences
// have fewer than kShortQueries queries on average: a pipeline's workgroup of 256 rows is
// mostly empty there.  Measured (us, short form against the pipeline), one MI355X: 197
// queries by 16 heads 11.4 and 17.7, 1024 19.8 and 37.6, 2048 47 and 63, 8 x 200 16.8 and
// 18.8, 256 x 1 51 and 154, 512 by 64 heads 23.4 and 26.5, 16 behind 4096 keys 53 and 82; 1350
// by 32 47.7 and 44.8, 2048 by 24 65 and 64, 1024 by 64 53 and 41, 4096 by 16 146 and 118.
// Beyond that many rows: 64 x 30 by 32 27 and 82, 500 x 20 behind 500 keys 919 and 1574, 256 x
// 64 by 16 144 and 203, but 128 x 64 behind 1000 403 and 338, 32 x 200 62 and 43.
// Behind a longer prefix every block of 32 queries reads it again, from the last-level cache or HBM where
// there are many K/V heads: then from 20 K rows on only sequences of one block stay with the short
// form.  With prefixes of 500, 1000, 4000 and 16000 keys: 1 x 192 by 128 32 45 140 619 and 30 41
// 108 386, 1 x 320 by 128 48 69 226 1027 and 34 52 134 502, 1 x 384 by 64 32 45 119 528 and 32 45 117
// 399, 4 x 100 by 64 42 74 310 1347 and 27 38 127 457, 16 x 64 by 32 52 92 368 1465 and 44 77 240 873,
// 64 x 40 by 32 207 378 1413 5692 and 199 315 969 3599.  On the other side of each limit: 8 x 32
// by 128 53 102 360 1402 and 93 153 487 1780, 10 x 64 by 32 36 58 228 930 and 42 61 222 811, 1 x
// 128 by 128 18 26 79 365 and 24 34 102 383, 1 x 2048 by 16 56 71 153 476 and 74 86 159 441; without a
// prefix 4 x 100 by 64 14 and 15, 16 x 64 by 32 14 and 24, 64 x 40 by 32 48 and 85.
static constexpr int64_t kShortRows = 40 * 1024, kShortQueries = 48;
static constexpr int64_t kPrefix = 500, kPrefixRows = 20 * 1024, kPrefixHeads = 64;

extern "C" int g9_latent_varlen_fwd(const void* q, const void* k, const void* v, const void* k_rope, void* o, float* lse,
                                    const int32_t* cu_q, const int32_t* cu_k, int64_t B, int64_t T, int64_t TK,
                                    int64_t HQ, int64_t HK, const int64_t* q_strides, const int64_t* k_strides,
                                    const int64_t* v_strides, int64_t k_rope_stride, const int64_t* o_strides,
                                    float sm_scale, int dtype, int causal, void* stream) {
  if (dtype != G9_F16 && dtype != G9_BF16) return G9_ERR_DTYPE;
  if (B < 0 || B > kMaxRows || T < 0 || T > kMaxRows || TK < 0 || TK > kMaxRows || HQ <= 0 || HQ > 65536 || HK <= 0 ||
      HQ % HK || !scale_ok(sm_scale))
    return G9_ERR_SHAPE;
  if (!q_strides || !k_strides || !v_strides || !o_strides) return G9_ERR_LAYOUT;
  // The step of a single row is never taken.
  const int64_t qs[2] = {T > 1 ? q_strides[0] : 192, HQ > 1 ? q_strides[1] : 0};
  const int64_t os[2] = {T > 1 ? o_strides[0] : 128, HQ > 1 ? o_strides[1] : 0};
  const int64_t ks[2] = {TK > 1 ? k_strides[0] : 128, HK > 1 ? k_strides[1] : 0};
  const int64_t vs[2] = {TK > 1 ? v_strides[0] : 128, HK > 1 ? v_strides[1] : 0};
  const int64_t rs[2] = {TK > 1 ? k_rope_stride : 64, 0};
  if (!steps(qs, 2) || !steps(ks, 2) || !steps(vs, 2) || !steps(rs, 2) || !steps(os, 2)) return G9_ERR_LAYOUT;
  const int64_t size[2] = {T, HQ};
  if (!apart(size, os, 2, 128)) return G9_ERR_LAYOUT;
  if (B == 0 || T == 0) return G9_OK;
  if (!q || !o || (TK && (!k || !v || !k_rope)) || !cu_q || !cu_k) return G9_ERR_LAYOUT;
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(k_rope) || !aligned16(o) || ((uintptr_t)lse & 3))
    return G9_ERR_LAYOUT;
  // Token strides within 32 bits, a tile's rows within a descriptor's range.
  for (const int64_t* st : {qs, ks, vs, rs, os})
    if (st[0] * 2 * fa::kBlockM >= (int64_t(1) << 31)) return G9_ERR_LAYOUT;
  fa::LatentVarParams p{};
  p.q = static_cast<const char*>(q);
  p.k = static_cast<const char*>(k);
  p.v = static_cast<const char*>(v);
  p.r = static_cast<const char*>(k_rope);
  p.o = static_cast<char*>(o);
  p.lse = lse;
  p.cu_q = cu_q;
  p.cu_k = cu_k;
  p.q_h = qs[1] * 2, p.k_h = ks[1] * 2, p.v_h = vs[1] * 2, p.o_h = os[1] * 2;
  p.ldq = (u32)(qs[0] * 2), p.ldk = (u32)(ks[0] * 2), p.ldv = (u32)(vs[0] * 2), p.ldr = (u32)(rs[0] * 2);
  p.ldo = (u32)(os[0] * 2);
  p.B = (int)B, p.T = (int)T, p.TK = (int)TK, p.HQ = (int)HQ, p.HK = (int)HK;
  p.causal = causal != 0;
  p.scale_log2 = sm_scale * fa::kLog2e;
  void* args[] = {&p};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const int64_t group = HQ / HK;
  const bool reread = B * HK >= kPrefixHeads && T * HQ > kPrefixRows && T > 32 * B && TK - T >= kPrefix * B;
  const bool few = (T * HQ <= kShortRows || T < kShortQueries * B) && !reread;
  if (few) {
    const int64_t blocks = T * group / 32 + (B < T ? B : T);
    if (blocks * HK * 256 > UINT32_MAX) return G9_ERR_SHAPE;  // the threads of a launch
    return launched(hipLaunchKernel(dtype == G9_BF16 ? reinterpret_cast<const void*>(g9_latent_varlen_short_bf16)
                                                     : reinterpret_cast<const void*>(g9_latent_varlen_short_f16),
                                    dim3((unsigned)(blocks * HK)), dim3(256), args, 0, st));
  }
  // At most T / 256 whole tiles and a partial one per sequence.
  const int64_t tiles = T / fa::kBlockM + (B < T ? B : T);
  const int64_t grid = 8 * group * ((tiles * HK + 7) / 8);
  if (grid * fa::kThreads > UINT32_MAX) return G9_ERR_SHAPE;  // the threads of a launch
  return launched(hipLaunchKernel(dtype == G9_BF16 ? reinterpret_cast<const void*>(g9_latent_varlen_bf16)
                                                   : reinterpret_cast<const void*>(g9_latent_varlen_f16),
                                  dim3((unsigned)grid), dim3(fa::kThreads), args, 0, st));
}
