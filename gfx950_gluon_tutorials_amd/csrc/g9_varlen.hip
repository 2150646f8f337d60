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

namespace g9 {
namespace fa {

// Few queries: a workgroup per 32 rows (queries by the query heads of a K/V head),
// its 4 waves taking the key tiles in turn and joining their sums in LDS; two
// workgroups a CU, so that one computes while the other waits for its tile (one,
// with two stages a wave: 66 us for 2048 queries instead of 38).  The pipeline's
// workgroups of 256 queries leave most of the chip idle there, and its 60 KB of code
// are fetched for a few tiles.
template <bool BF16, int HD>
struct ShortWave {
  using T = Wave<VarParams, BF16, HD, 1, 1>;
  static constexpr int kLds = 4 * T::kWaveLds;
};
template <bool BF16, int HD>
G9_DEV void varlen_short(const VarParams& p, char* smem) {
  using W = typename ShortWave<BF16, HD>::T;
  const int group = p.HQ / p.HK;
  const int rank = blockIdx.x / p.HK, hk = blockIdx.x - rank * p.HK;
  Tile t;
  if (!find_tile<32, 256>(p, rank, group, reinterpret_cast<int*>(smem), t)) return;
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  W w(p);
  w.init(smem, wave, p.ldk, p.ldv);
  const int row = t.mb * 32 + w.col, nd = row / group, hq = hk * group + row - nd * group;
  const bool in = nd < t.lq;
  w.node[0] = in ? nd : -1;
  w.context = p.causal ? t.lk - t.lq : t.lk;
  w.q0 = t.q0, w.keys = t.lk;
  // The first row of the block reads the keys below `all`, the last one those
  // below `need`.
  const int last = min((t.mb * 32 + 31) / group, t.lq - 1);
  const int need = uniform(min(max(last + 1 + w.context, 0), t.lk));
  const int all = uniform(min(max(t.mb * 32 / group + 1 + w.context, 0), t.lk));
  const char* const kp = p.k + hk * p.k_h + (size_t)t.k0 * p.ldk;
  const char* const vp = p.v + hk * p.v_h + (size_t)t.k0 * p.ldv;
  const auto fill = [&](int tile) {
#pragma unroll
    for (int i = 0; i < W::kPieces; ++i) {
      const int k = tile * W::kKeys + 16 * i;
      w.fill_piece(i, 0, kp + (size_t)(u32)k * p.ldk, vp + (size_t)(u32)k * p.ldv, min(max(t.lk - k, 0), 16), p.ldk,
                   p.ldv);
    }
  };
  const int tiles = (need + W::kKeys - 1) / W::kKeys;
  if (wave < tiles) fill(wave);
  w.load_q(0, p.q + (size_t)(t.q0 + (in ? nd : 0)) * p.ldq + (in ? hq : hk * group) * p.q_h);
  w.clear();
  for (int i = wave; i < tiles; i += 4) {
    waitcnt<0, 0>();
    __builtin_amdgcn_sched_barrier(0);
    w.tile(i * W::kKeys, 0, (i + 1) * W::kKeys > all);
    waitcnt<63, 0>();
    __builtin_amdgcn_sched_barrier(0);
    if (i + 4 < tiles) fill(i + 4);
  }
  // The waves' sums, each in its own stage: rows 16 bytes more than HD floats
  // apart (banks), behind them maximum and weight.
  constexpr int kPitch = HD + 4, kSums = 32 * kPitch;
  static_assert((kSums + 64) * 4 <= W::kWaveLds);
  const float lw = xhalf(w.l[0], [](float x, float y) { return x + y; });
  waitcnt<63, 0>();
  const auto sums = [&](int i) { return reinterpret_cast<float*>(smem + i * W::kWaveLds); };
#pragma unroll
  for (int d = 0; d < W::kND; ++d)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      *reinterpret_cast<f32x4*>(sums(wave) + w.col * kPitch + 32 * d + 8 * r + 4 * w.h) =
          f32x4{w.o[0][d][4 * r], w.o[0][d][4 * r + 1], w.o[0][d][4 * r + 2], w.o[0][d][4 * r + 3]};
  if (w.h == 0) sums(wave)[kSums + w.col] = w.m[0], sums(wave)[kSums + 32 + w.col] = lw;
  __syncthreads();
  // Eight threads a row.
  const int r = tid >> 3, c = tid & 7, mine = t.mb * 32 + r, n = mine / group;
  if (n >= t.lq) return;
  float m = sums(0)[kSums + r];
#pragma unroll
  for (int i = 1; i < 4; ++i) m = __builtin_fmaxf(m, sums(i)[kSums + r]);
  float f[4], l = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[i] = __builtin_amdgcn_exp2f(sums(i)[kSums + r] - m);
    l += f[i] * sums(i)[kSums + 32 + r];
  }
  const bool none = (__float_as_uint(l) << 1) == 0;
  const float inv = none ? 0.f : 1.f / l;
  const int head = hk * group + mine - n * group;
  char* const orow = p.o + head * p.o_h + (size_t)(t.q0 + n) * p.ldo;
#pragma unroll
  for (int j = 0; j < HD / 32; ++j) {
    const int col = 32 * j + 4 * c;
    f32x4 x = {};
#pragma unroll
    for (int i = 0; i < 4; ++i) x += f[i] * *reinterpret_cast<const f32x4*>(sums(i) + r * kPitch + col);
    *reinterpret_cast<u32x2*>(orow + col * 2) = u32x2{pack2<BF16>(x[0] * inv, x[1] * inv), pack2<BF16>(x[2] * inv, x[3] * inv)};
  }
  if (p.lse && c == 0) p.lse[(size_t)head * p.T + t.q0 + n] = none ? -__builtin_inff() : (m + __builtin_log2f(l)) * kLn2;
}

}  // namespace fa
}  // namespace g9

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
    __shared__ __attribute__((aligned(1024))) char smem[fa::ShortWave<BF16, HD>::kLds];      \
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
