// Flash-attention forward over packed sequences of different lengths, causal or
// not (g9_varlen_fwd, include/gfx950_fmha.h), on the pipeline of
// g9_fmha_pipe.hpp: one workgroup per 256 queries of one sequence and head, its 8
// waves 32 queries each, walking the keys that the last of them may read.
//
// Bound by the matrix unit (4 D flops a query and key).  A causal row tile's
// cost grows with its place in its sequence, so the tiles of the whole batch are
// dispatched in the order of falling cost: the last workgroups to start are
// the shortest, and a batch of uneven prompts leaves no long tail.  Which tile
// a workgroup takes follows from the lengths alone and is worked out by the
// workgroup itself (find_tile), so no launch comes before this one and no
// length reaches the host.
#include "../../include/gfx950_fmha.h"
#include "g9_attn_host.hpp"
#include "g9_packed.hpp"

using namespace g9;
using namespace g9::host;

#define G9_VARLEN_KERNEL(NAME, BF16, HD)                                                                   \
  extern "C" __global__ __launch_bounds__(fa::kThreads) __attribute__((amdgpu_waves_per_eu(2, 2))) void \
  NAME(fa::VarParams p) {                                                                                 \
    __shared__ __attribute__((aligned(1024))) char smem[fa::VarPipe<fa::VarParams, BF16, HD>::kLds];                      \
    fa::varlen_fwd<BF16, HD>(p, smem);                                                                    \
  }
#define G9_SHORT_KERNEL(NAME, BF16, HD)                                                     \
  extern "C" __global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) void \
  NAME(fa::VarParams p) {                                                                   \
    __shared__ __attribute__((aligned(1024))) char smem[fa::ShortWave<fa::VarParams, BF16, HD>::kLds];      \
    fa::varlen_short<BF16, HD>(p, smem);                                                    \
  }
G9_SHORT_KERNEL(g9_varlen_short_bf16, true, 128)
G9_SHORT_KERNEL(g9_varlen_short_f16, false, 128)
G9_SHORT_KERNEL(g9_varlen_short_bf16_d64, true, 64)
G9_SHORT_KERNEL(g9_varlen_short_f16_d64, false, 64)
G9_VARLEN_KERNEL(g9_varlen_bf16, true, 128)
G9_VARLEN_KERNEL(g9_varlen_f16, false, 128)
G9_VARLEN_KERNEL(g9_varlen_bf16_d64, true, 64)
G9_VARLEN_KERNEL(g9_varlen_f16_d64, false, 64)

// Up to this many rows (queries by query heads) the short form runs.  Measured
// (us, short form against the pipeline; 16 heads of 128 where not said), one
// MI355X: 197 queries 7.2 and 16.8, 1024 17.3 and 32.9, 2048 38 and 56, 8 x 200
// 15.7 and 18.1, 256 x 1 13 and 139, 512 by 64 heads 20.8 and 24.0, 1350 by 32
// 31.7 and 34.5; behind it 32 x 200 47 and 41, 4096 121 and 107, 1024 by 64 51 and
// 39.
static constexpr int64_t kShortRows = 48 * 1024;

extern "C" int g9_varlen_fwd(const void* q, const void* k, const void* v, void* o, float* lse, const int32_t* cu_q,
                  const int32_t* cu_k, int64_t B, int64_t T, int64_t TK, int64_t HQ, int64_t HK, int64_t D,
                  const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides,
                  const int64_t* o_strides, float sm_scale, int dtype, int causal, void* stream) {
  if (dtype != G9_F16 && dtype != G9_BF16) return G9_ERR_DTYPE;
  if (B < 0 || B > kMaxRows || T < 0 || T > kMaxRows || TK < 0 || TK > kMaxRows || HQ <= 0 || HQ > 65536 || HK <= 0 ||
      HQ % HK || (D != 64 && D != 128) || !scale_ok(sm_scale))
    return G9_ERR_SHAPE;
  if (!q_strides || !k_strides || !v_strides || !o_strides) return G9_ERR_LAYOUT;
  // The step of a single row is never taken.
  const int64_t qs[2] = {T > 1 ? q_strides[0] : D, q_strides[1]}, os[2] = {T > 1 ? o_strides[0] : D, o_strides[1]};
  const int64_t ks[2] = {TK > 1 ? k_strides[0] : D, k_strides[1]}, vs[2] = {TK > 1 ? v_strides[0] : D, v_strides[1]};
  if (!steps(qs, 2) || !steps(ks, 2) || !steps(vs, 2) || !steps(os, 2)) return G9_ERR_LAYOUT;
  const int64_t size[2] = {T, HQ};
  if (!apart(size, os, 2, D)) return G9_ERR_LAYOUT;
  if (B == 0 || T == 0) return G9_OK;
  if (!q || !o || (TK && (!k || !v)) || !cu_q || !cu_k) return G9_ERR_LAYOUT;
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(o) || ((uintptr_t)lse & 3)) return G9_ERR_LAYOUT;
  // Token strides within 32 bits, a tile's rows within a descriptor's range.
  for (const int64_t* st : {qs, ks, vs, os})
    if (st[0] * 2 * fa::kBlockM >= (int64_t(1) << 31)) return G9_ERR_LAYOUT;
  fa::VarParams p{};
  p.q = static_cast<const char*>(q);
  p.k = static_cast<const char*>(k);
  p.v = static_cast<const char*>(v);
  p.o = static_cast<char*>(o);
  p.lse = lse;
  p.cu_q = cu_q;
  p.cu_k = cu_k;
  p.q_h = qs[1] * 2, p.k_h = ks[1] * 2, p.v_h = vs[1] * 2, p.o_h = os[1] * 2;
  p.ldq = (u32)(qs[0] * 2), p.ldk = (u32)(ks[0] * 2), p.ldv = (u32)(vs[0] * 2), p.ldo = (u32)(os[0] * 2);
  p.B = (int)B, p.T = (int)T, p.TK = (int)TK, p.HQ = (int)HQ, p.HK = (int)HK;
  p.causal = causal != 0;
  p.scale_log2 = sm_scale * fa::kLog2e;
  void* args[] = {&p};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const int64_t group = HQ / HK;
  if (T * HQ <= kShortRows) {
    const int64_t blocks = T * group / 32 + (B < T ? B : T);
    static const void* const kShort[2][2] = {
        {reinterpret_cast<const void*>(g9_varlen_short_f16), reinterpret_cast<const void*>(g9_varlen_short_bf16)},
        {reinterpret_cast<const void*>(g9_varlen_short_f16_d64), reinterpret_cast<const void*>(g9_varlen_short_bf16_d64)}};
    return launched(hipLaunchKernel(kShort[D == 64][dtype == G9_BF16], dim3((unsigned)(blocks * HK)), dim3(256), args, 0, st));
  }
  // At most T / 256 whole tiles and a partial one per sequence.
  const int64_t tiles = T / fa::kBlockM + (B < T ? B : T);
  const int64_t grid = 8 * group * ((tiles * HK + 7) / 8);
  if (grid * fa::kThreads > UINT32_MAX) return G9_ERR_SHAPE;  // the threads of a launch
  static const void* const kFns[2][2] = {
      {reinterpret_cast<const void*>(g9_varlen_f16), reinterpret_cast<const void*>(g9_varlen_bf16)},
      {reinterpret_cast<const void*>(g9_varlen_f16_d64), reinterpret_cast<const void*>(g9_varlen_bf16_d64)}};
  return launched(hipLaunchKernel(kFns[D == 64][dtype == G9_BF16], dim3((unsigned)grid), dim3(fa::kThreads), args, 0, st));
}
