// Attention over a paged cache of latents (g9_latent_fwd, include/gfx950_fmha.h):
// a token's row holds one latent of 512 values, which is every head's value and the
// larger part of its key, and a rotated key of 64 that the heads share too.
#include "../../include/gfx950_fmha.h"
#include "g9_attn_host.hpp"
#include "g9_line.hpp"

namespace g9 {
namespace latent {

using namespace fa;

constexpr int kRank = 512, kRow = 576;  // values of a latent, of a row

struct Params {
  const char* q;
  const char* cache;
  char* o;
  float* lse;                                      // [H][T], or null
  const int* table;
  const int* lengths;
  const int* cu;
  const unsigned long long* mask;                  // or null: a chain
  long long q_t, q_h, o_t, o_h;                    // token / head strides, bytes
  long long c_b, c_t;                              // block / token strides, bytes
  long long table_stride;
  int num_blocks, width, shift, words;
  int B, T, H;
  float scale_log2;
};

// A wave per query and head: lane i has the values 8 i .. 8 i + 7 and 512 + i of a
// row, a key at a time.
template <bool BF16>
G9_DEV void plain_fwd(const Params& p) {
  const int lane = threadIdx.x & 63;
  const long long w = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int t = (int)(w / p.H), h = (int)(w - (long long)t * p.H);
  if (t >= p.T) return;
  int b = -1, q0 = 0, n = 0;
  for (int i = 0; i < p.B; ++i) {
    q0 = min(max(p.cu[i], 0), p.T);
    n = min(max(p.cu[i + 1], q0), p.T) - q0;
    if (t >= q0 && t < q0 + n) {
      b = i;
      break;
    }
  }
  if (b < 0) return;
  const NodeRow row = {t - q0, max(p.lengths[b], 0), q0};
  const int keys = (int)min((long long)row.context + n, (long long)p.width << p.shift);
  const auto load = [&](const char* r, float (&x)[9]) {
    const u32x4 a = *reinterpret_cast<const u32x4*>(r + lane * 16);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const f32x2 v = unpack2<BF16>(a[e]);
      x[2 * e] = v.x, x[2 * e + 1] = v.y;
    }
    x[8] = unpack2<BF16>(*reinterpret_cast<const uint16_t*>(r + kRank * 2 + lane * 2)).x;
  };
  float q[9], o[8] = {}, m = -3.0e38f, l = 0.f;
  load(p.q + t * p.q_t + h * p.q_h, q);
  for (int k0 = 0; k0 < keys; k0 += 64) {
    const unsigned long long reads = node_reads(p, row, k0, keys);
    for (int i = 0; i < 64; ++i) {
      if (!(reads >> i & 1)) continue;
      const int k = k0 + i, page = p.table[b * p.table_stride + (k >> p.shift)];
      float x[9] = {};
      if ((u32)page < (u32)p.num_blocks)
        load(p.cache + page * p.c_b + (unsigned long long)(k & ((1 << p.shift) - 1)) * p.c_t, x);
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < 9; ++e) s = __builtin_fmaf(q[e], x[e], s);
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) s += __shfl_xor(s, d, 64);
      s *= p.scale_log2;
      const float m_new = __builtin_fmaxf(m, s), f = __builtin_amdgcn_exp2f(m - m_new), g = __builtin_amdgcn_exp2f(s - m_new);
      l = l * f + g;
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = o[e] * f + g * x[e];
      m = m_new;
    }
  }
  const bool none = l == 0.f;
  const float inv = none ? 0.f : 1.f / l;
  u32x4 out;
#pragma unroll
  for (int e = 0; e < 4; ++e) out[e] = pack2<BF16>(o[2 * e] * inv, o[2 * e + 1] * inv);
  *reinterpret_cast<u32x4*>(p.o + t * p.o_t + h * p.o_h + lane * 16) = out;
  if (p.lse && lane == 0) p.lse[(long long)h * p.T + t] = none ? -__builtin_inff() : (m + __builtin_log2f(l)) * kLn2;
}

}  // namespace latent
}  // namespace g9

using namespace g9;
using namespace g9::host;

extern "C" __global__ __launch_bounds__(256) void g9_latent_bf16(latent::Params p) { latent::plain_fwd<true>(p); }
extern "C" __global__ __launch_bounds__(256) void g9_latent_f16(latent::Params p) { latent::plain_fwd<false>(p); }

extern "C" size_t g9_latent_workspace_size(int64_t B, int64_t T, int64_t H) {
  if (B <= 0 || T <= 0 || H <= 0) return 0;
  return 32;
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
  p.q_t = qs[0] * 2, p.q_h = qs[1] * 2, p.o_t = os[0] * 2, p.o_h = os[1] * 2;
  p.c_b = cs[0] * 2, p.c_t = cs[1] * 2;
  p.table_stride = table_stride;
  p.num_blocks = (int)num_blocks, p.width = (int)width, p.shift = log2_of(block_size), p.words = (int)words;
  p.B = (int)B, p.T = (int)T, p.H = (int)H;
  p.scale_log2 = sm_scale * fa::kLog2e;
  void* args[] = {&p};
  return launched(hipLaunchKernel(dtype == G9_BF16 ? reinterpret_cast<const void*>(g9_latent_bf16)
                                                   : reinterpret_cast<const void*>(g9_latent_f16),
                                  dim3((unsigned)((T * H + 3) / 4)), dim3(256), args, 0,
                                  reinterpret_cast<hipStream_t>(stream)));
}
