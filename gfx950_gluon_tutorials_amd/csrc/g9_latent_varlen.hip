// Attention over packed sequences whose keys and values were expanded from
// latents (g9_latent_varlen_fwd, include/gfx950_fmha.h): a head's key is 128 values
// of its own and 64 rotated ones that all heads share, its value 128.
#include "../../include/gfx950_fmha.h"
#include "g9_attn_host.hpp"
#include "g9_wave.hpp"

namespace g9 {
namespace fa {

struct LatentVarParams {
  const char* q;
  const char* k;
  const char* v;
  const char* r;                               // the shared keys
  char* o;
  float* lse;                                  // [HQ][T] fp32, or null
  const int* cu_q;
  const int* cu_k;
  long long q_h, k_h, v_h, o_h;                // head strides, bytes
  u32 ldq, ldk, ldv, ldr, ldo;                 // token strides, bytes
  int B, T, TK, HQ, HK, causal;
  float scale_log2;
};

// A wave per query and head, a key at a time: lane i has the values 2 i and 2 i + 1
// of a head's own key and value, and 128 + i of the shared one.
template <bool BF16>
G9_DEV void latent_varlen_plain(const LatentVarParams& p) {
  const int lane = threadIdx.x & 63;
  const long long w = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int t = (int)(w / p.HQ), h = (int)(w - (long long)t * p.HQ), hk = h / (p.HQ / p.HK);
  if (t >= p.T) return;
  int b = -1, q0 = 0, lq = 0;
  for (int i = 0; i < p.B; ++i) {
    q0 = min(max(p.cu_q[i], 0), p.T);
    lq = min(max(p.cu_q[i + 1], q0), p.T) - q0;
    if (t >= q0 && t < q0 + lq) {
      b = i;
      break;
    }
  }
  if (b < 0) return;
  const int k0 = min(max(p.cu_k[b], 0), p.TK), lk = min(max(p.cu_k[b + 1], k0), p.TK) - k0;
  const int end = p.causal ? min(t - q0 + 1 + lk - lq, lk) : lk;
  const auto two = [&](const char* at) { return unpack2<BF16>(*reinterpret_cast<const u32*>(at + lane * 4)); };
  const auto one = [&](const char* at) { return unpack2<BF16>(*reinterpret_cast<const uint16_t*>(at + lane * 2)).x; };
  const char* const q = p.q + (long long)t * p.ldq + h * p.q_h;
  const f32x2 qn = two(q);
  const float qr = one(q + 256);
  f32x2 o = {0.f, 0.f};
  float m = -3.0e38f, l = 0.f;
  for (int j = k0; j < k0 + end; ++j) {
    const f32x2 kn = two(p.k + (long long)j * p.ldk + hk * p.k_h), x = two(p.v + (long long)j * p.ldv + hk * p.v_h);
    float s = qn.x * kn.x + qn.y * kn.y + qr * one(p.r + (long long)j * p.ldr);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) s += __shfl_xor(s, d, 64);
    s *= p.scale_log2;
    const float m_new = __builtin_fmaxf(m, s), f = __builtin_amdgcn_exp2f(m - m_new), g = __builtin_amdgcn_exp2f(s - m_new);
    l = l * f + g;
    o.x = o.x * f + g * x.x, o.y = o.y * f + g * x.y;
    m = m_new;
  }
  const bool none = l == 0.f;
  const float inv = none ? 0.f : 1.f / l;
  *reinterpret_cast<u32*>(p.o + (long long)t * p.ldo + h * p.o_h + lane * 4) = pack2<BF16>(o.x * inv, o.y * inv);
  if (p.lse && lane == 0) p.lse[(long long)h * p.T + t] = none ? -__builtin_inff() : (m + __builtin_log2f(l)) * kLn2;
}

}  // namespace fa
}  // namespace g9

using namespace g9;
using namespace g9::host;

extern "C" __global__ __launch_bounds__(256) void g9_latent_varlen_bf16(fa::LatentVarParams p) {
  fa::latent_varlen_plain<true>(p);
}
extern "C" __global__ __launch_bounds__(256) void g9_latent_varlen_f16(fa::LatentVarParams p) {
  fa::latent_varlen_plain<false>(p);
}

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
  const int64_t waves = T * HQ;
  if ((waves + 3) / 4 * 256 > UINT32_MAX) return G9_ERR_SHAPE;  // the threads of a launch
  void* args[] = {&p};
  return launched(hipLaunchKernel(dtype == G9_BF16 ? reinterpret_cast<const void*>(g9_latent_varlen_bf16)
                                                   : reinterpret_cast<const void*>(g9_latent_varlen_f16),
                                  dim3((unsigned)((waves + 3) / 4)), dim3(256), args, 0,
                                  reinterpret_cast<hipStream_t>(stream)));
}
