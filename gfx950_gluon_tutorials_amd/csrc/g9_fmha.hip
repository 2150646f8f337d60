// Flash-attention forward (non-causal) for gfx950: O = softmax(Q K^T * sm_scale) V
// per (batch, query head), with grouped K/V heads (query head h reads K/V head
// h * HK / HQ).  Head dim 128 or 64, FP16 or BF16 in and out, fp32 softmax
// and accumulation.  extern "C" entry: g9_fmha_fwd (include/gfx950_fmha.h).
//
// One workgroup owns 256 query rows of one (batch, head) and walks all keys in
// tiles of 8192 / D keys (64 at head dim 128, 128 at 64).  Its 8 waves (2 per
// SIMD) own 32 query rows each, so every row-wise reduction stays inside a
// wave.  Per key tile a wave runs
//   S^T = K . Q^T    16 MFMAs 32x32x16 (32-key blocks x D/16 steps of 16 d);
//                    K fragments from LDS, Q fragments in registers;
//   online softmax   running max m and (lane-partial) sum l in log2 units;
//   O^T += V^T . P^T 16 MFMAs (D/32 blocks of 32 d x steps of 16 keys);
//                    P^T straight from the S^T registers, V^T through LDS
//                    transpose reads.
// The scores are computed transposed (the keys are the MFMA's rows): lane l
// then holds 16 keys of query l % 32 per 32-key block, so the row max and
// the row sum of a query are in-lane reductions plus one exchange with lane
// l ^ 32, the accumulator rescale is one per-lane factor, and the score
// registers are already the B operand of the PV MFMA once its 16-key steps use
// the key order the score layout gives each lane half: step t, lane half h,
// slot u covers key 16t + 8(u / 4) + 4h + (u % 4).  V is read in that key order
// with ds_read_b64_tr_b16, which within each 16-lane group gives lane 4a + b
// element b of the 8-byte rows addressed by lanes a, a + 4, a + 8, a + 12
// (measured on gfx950): 4 keys of one head-dim column per read.
//
// The loop is software pipelined over four clusters with the two waves of a
// SIMD one cluster apart (see Pipe in g9_fmha_pipe.hpp).
#include <stdint.h>

#include "../../include/gfx950_fmha.h"
#include "g9_fmha_pipe.hpp"

namespace g9 {
namespace fa {

// Optional phase stamps (build with -DG9_TIMING; read by profiling.py through
// g9_fmha_timing_read): thread 0 of each workgroup records s_memtime (shader
// clock) and s_memrealtime (100 MHz) at kernel entry, loop start, loop end and
// kernel end, for the first kTimingWorkgroups workgroups (by block index).
// Each stamp waits only for its own scalar reads.  Nothing in the regular
// build.
#ifdef G9_TIMING
constexpr int kTimingWorkgroups = 16384;
__device__ unsigned long long g9_fmha_timing_buf[kTimingWorkgroups * 8];
G9_DEV void stamp(int slot) {
  __builtin_amdgcn_sched_barrier(0);
  const unsigned long long t = __builtin_amdgcn_s_memtime();
  const unsigned long long r = __builtin_amdgcn_s_memrealtime();
  __builtin_amdgcn_s_waitcnt((63 & 15) | (7 << 4) | (0 << 8) | ((63 >> 4) << 14));  // lgkmcnt(0) only
  if (threadIdx.x == 0 && blockIdx.x < kTimingWorkgroups) {
    g9_fmha_timing_buf[blockIdx.x * 8 + slot * 2] = t;
    g9_fmha_timing_buf[blockIdx.x * 8 + slot * 2 + 1] = r;
  }
  __builtin_amdgcn_sched_barrier(0);
}
#else
G9_DEV void stamp(int) {}
#endif

struct FaParams {
  const char* q;
  const char* k;
  const char* v;
  char* o;
  float* lse;                        // [B][HQ][S] fp32, or null
  long long q_b, q_h, k_b, k_h, v_b, v_h, o_b, o_h;  // batch / head strides, bytes
  u32 ldq, ldk, ldv, ldo;            // sequence strides, bytes
  int B, HQ, HK, S;
  int mblocks;                       // ceil(S / 256)
  int num_xcds;
  float scale_log2;                  // sm_scale * log2(e)
  int scale_on_q;                    // fold scale_log2 into Q (rounded to 16 bit) before the loop
};

// smem: PipeT::kLdsBytes of LDS, 1024-byte aligned, declared by the kernel
// (one array for both scale placements a kernel instantiates).
template <bool BF16, bool LAZY, bool SOQ, int HD>
G9_DEV void fmha_fwd(const FaParams& p, char* smem) {
  using PipeT = Pipe<FaParams, BF16, LAZY, SOQ, HD>;
  stamp(0);
  const int total = p.B * p.HQ * p.mblocks;
  int pid, unused;
  tile_coords(blockIdx.x, total, total, 1, p.num_xcds, 1, pid, unused);
  const int bh = pid / p.mblocks, mb = pid - bh * p.mblocks;
  const int b = bh / p.HQ, hq = bh - b * p.HQ;
  const int hk = hq * p.HK / p.HQ;
  const int tid = threadIdx.x, lane = tid & 63;
  const int h = lane >> 5;

  PipeT P(p);
  P.wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  P.nt = (p.S + PipeT::kBN - 1) / PipeT::kBN;
  P.nte = (P.nt + 1) & ~1;
  P.nfull = p.S / PipeT::kBN;
  P.lds0 = (u32)(uintptr_t)to_lds(smem);
  const int nte = P.nte, wave = P.wave;
  const char* qb = p.q + b * p.q_b + hq * p.q_h;
  const rsrc_t rq = make_rsrc(qb, (u32)p.S * p.ldq);
  P.rk = make_rsrc(p.k + b * p.k_b + hk * p.k_h, (u32)p.S * p.ldk);
  P.rv = make_rsrc(p.v + b * p.v_b + hk * p.v_h, (u32)p.S * p.ldv);

  const int qrow = mb * kBlockM + wave * 32 + (lane & 31);
#pragma unroll
  for (int s = 0; s < PipeT::kNS; ++s)
    P.qf[s] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rq, (u32)qrow * p.ldq + (16 * s + 8 * h) * 2, 0, 0));
  P.voffk = (u32)lane * p.ldk;
  P.voffv = (u32)lane * p.ldv;
  P.ak = P.lds0 + h * PipeT::kPitchK + (lane & 31) * 16;
  {
    const int G = lane >> 4, jj = lane & 15;
    P.av = P.lds0 + PipeT::kLdsV + (2 * (G & 1) + ((jj & 3) >> 1)) * PipeT::kPitchV + (4 * (G >> 1) + (jj >> 2)) * 16 +
           8 * (jj & 1);
  }
  // Prologue: K_0, V_0, K_1 in; S_0 and its first softmax half; K_2 and V_1
  // requested (in that order: the loop expects K_{j+2} before V_{j+1}); K_1
  // in registers.
  P.dma_k(0, 0);
  P.dma_v(0, 0);
  P.dma_k(1, 1);
  P.sc = p.scale_log2;
  if constexpr (SOQ) {
#pragma unroll
    for (int s = 0; s < PipeT::kNS; ++s)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const f32x2 x = unpack2<BF16>(P.qf[s][e]);
        P.qf[s][e] = pack2<BF16>(x.x * P.sc, x.y * P.sc);
      }
    P.sc = 1.f;
  }
#pragma unroll
  for (int d = 0; d < PipeT::kND; ++d) P.o[d] = f32x16{};
  P.m = -__builtin_inff();
  P.l = 0.f;
  waitcnt<0, 15>();
  barrier();
  P.template read_k<0>();
  typename PipeT::Sc sa, sb;
  P.qk(sa);
  waitcnt<63, 0>();
  barrier();  // every wave has read K_0: its buffer takes K_2
  if (nte > 2) P.dma_k(2, 0);
  P.dma_v(1, 1);
  if (p.S < PipeT::kBN) P.mask(sa, p.S);  // tile 0 itself ends early
  P.vec0(sa);
  P.vec1(sa);
  P.l *= P.alpha;
  P.template read_k<1>();
  waitcnt<63, 0>();

  const bool lag = wave >= 4;
  stamp(1);
  if (lag) barrier();
  int j = 0;
  for (; j + 2 < nte; j += 2) {
    P.template step<0, true>(j, sa, sb);
    P.template step<1, true>(j + 1, sb, sa);
  }
  P.template step<0, true>(j, sa, sb);
  P.template step<1, false>(j + 1, sb, sa);
  __builtin_amdgcn_s_setprio(0);
  if (!lag) barrier();
  stamp(2);

  const float lt = xhalf(P.l, [](float x, float y) { return x + y; });
  const float inv = 1.f / lt;
  if (qrow < p.S) {
    char* orow = p.o + b * p.o_b + hq * p.o_h + (size_t)qrow * p.ldo;
#pragma unroll
    for (int d = 0; d < PipeT::kND; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int col = 32 * d + 8 * r + 4 * h;
        const u32x2 w = {pack2<BF16>(P.o[d][4 * r] * inv, P.o[d][4 * r + 1] * inv),
                         pack2<BF16>(P.o[d][4 * r + 2] * inv, P.o[d][4 * r + 3] * inv)};
        *reinterpret_cast<u32x2*>(orow + col * 2) = w;
      }
    if (p.lse && h == 0) p.lse[((size_t)b * p.HQ + hq) * p.S + qrow] = (P.m + __builtin_log2f(lt)) * kLn2;
  }
  stamp(3);
}

}  // namespace fa
}  // namespace g9

using namespace g9;

// Kernels: g9_fmha_fwd_{bf16,f16}_v{3,4}[_d64]; v3 rescales every tile, v4
// lazily; head dim 128, or 64 with the _d64 suffix.
#define G9_FMHA_KERNEL(NAME, BF16, LAZY, HD)                                                              \
  extern "C" __global__ __launch_bounds__(fa::kThreads) __attribute__((amdgpu_waves_per_eu(2, 2))) void \
  NAME(fa::FaParams p) {                                                                                  \
    __shared__ __attribute__((aligned(1024))) char smem[fa::Pipe<fa::FaParams, BF16, LAZY, true, HD>::kLdsBytes];        \
    if (p.scale_on_q)                                                                                     \
      fa::fmha_fwd<BF16, LAZY, true, HD>(p, smem);                                                        \
    else                                                                                                  \
      fa::fmha_fwd<BF16, LAZY, false, HD>(p, smem);                                                       \
  }
G9_FMHA_KERNEL(g9_fmha_fwd_bf16_v3, true, false, 128)
G9_FMHA_KERNEL(g9_fmha_fwd_f16_v3, false, false, 128)
G9_FMHA_KERNEL(g9_fmha_fwd_bf16_v4, true, true, 128)
G9_FMHA_KERNEL(g9_fmha_fwd_f16_v4, false, true, 128)
G9_FMHA_KERNEL(g9_fmha_fwd_bf16_v3_d64, true, false, 64)
G9_FMHA_KERNEL(g9_fmha_fwd_f16_v3_d64, false, false, 64)
G9_FMHA_KERNEL(g9_fmha_fwd_bf16_v4_d64, true, true, 64)
G9_FMHA_KERNEL(g9_fmha_fwd_f16_v4_d64, false, true, 64)

extern "C" int g9_fmha_fwd(const void* q, const void* k, const void* v, void* o, float* lse, int64_t B, int64_t HQ,
                           int64_t HK, int64_t S, int64_t D, const int64_t* q_strides, const int64_t* k_strides,
                           const int64_t* v_strides, const int64_t* o_strides, float sm_scale, int dtype,
                           int scale_on_q, int variant, void* stream) {
  if (dtype != G9_F16 && dtype != G9_BF16) return G9_ERR_DTYPE;
  if (variant != 3 && variant != 4) return G9_ERR_SCHEDULE;
  if (B <= 0 || HQ <= 0 || HK <= 0 || S <= 0 || HQ % HK != 0) return G9_ERR_SHAPE;
  if ((D != 128 && D != 64) || S % 64 != 0) return G9_ERR_SHAPE;
  if (!q || !k || !v || !o || !q_strides || !k_strides || !v_strides || !o_strides) return G9_ERR_LAYOUT;
  const int64_t* st[4] = {q_strides, k_strides, v_strides, o_strides};
  const void* ptr[4] = {q, k, v, o};
  for (int i = 0; i < 4; ++i) {
    // (batch, head, seq, dim) strides in elements: unit head-dim stride,
    // 16-byte aligned rows, and every row offset of a (batch, head) slice,
    // including a 256-row tile past the end, inside 31 bits.
    if (st[i][3] != 1 || st[i][2] < D || (st[i][2] * 2) % 16 != 0 || st[i][0] < 0 || st[i][1] < 0) return G9_ERR_LAYOUT;
    if ((uintptr_t)ptr[i] % 16 != 0 || (st[i][0] * 2) % 16 != 0 || (st[i][1] * 2) % 16 != 0) return G9_ERR_LAYOUT;
    if ((S + fa::kBlockM) * st[i][2] * 2 >= (int64_t(1) << 31)) return G9_ERR_SHAPE;
  }
  if (lse && (uintptr_t)lse % 4 != 0) return G9_ERR_LAYOUT;
  const int64_t mblocks = (S + fa::kBlockM - 1) / fa::kBlockM;
  if (B * HQ * mblocks > INT32_MAX) return G9_ERR_SHAPE;
  // This file is compiled without NaN semantics (-fno-honor-nans), under
  // which a float comparison may treat NaN as ordered: the scale's bits are
  // tested instead (a positive, finite, nonzero float).
  const u32 sm_bits = __builtin_bit_cast(u32, sm_scale);
  if ((sm_bits >> 31) != 0 || sm_bits == 0 || ((sm_bits >> 23) & 0xff) == 0xff) return G9_ERR_SHAPE;
  fa::FaParams p{};
  p.q = static_cast<const char*>(q);
  p.k = static_cast<const char*>(k);
  p.v = static_cast<const char*>(v);
  p.o = static_cast<char*>(o);
  p.lse = lse;
  p.q_b = q_strides[0] * 2;
  p.q_h = q_strides[1] * 2;
  p.k_b = k_strides[0] * 2;
  p.k_h = k_strides[1] * 2;
  p.v_b = v_strides[0] * 2;
  p.v_h = v_strides[1] * 2;
  p.o_b = o_strides[0] * 2;
  p.o_h = o_strides[1] * 2;
  p.ldq = (u32)(q_strides[2] * 2);
  p.ldk = (u32)(k_strides[2] * 2);
  p.ldv = (u32)(v_strides[2] * 2);
  p.ldo = (u32)(o_strides[2] * 2);
  p.B = (int)B;
  p.HQ = (int)HQ;
  p.HK = (int)HK;
  p.S = (int)S;
  p.mblocks = (int)mblocks;
  p.num_xcds = 8;
  p.scale_log2 = sm_scale * fa::kLog2e;
  p.scale_on_q = scale_on_q != 0;
  void* args[] = {&p};
  // [head dim 64][lazy][bf16]
  static const void* const kFns[2][2][2] = {
      {{reinterpret_cast<const void*>(g9_fmha_fwd_f16_v3), reinterpret_cast<const void*>(g9_fmha_fwd_bf16_v3)},
       {reinterpret_cast<const void*>(g9_fmha_fwd_f16_v4), reinterpret_cast<const void*>(g9_fmha_fwd_bf16_v4)}},
      {{reinterpret_cast<const void*>(g9_fmha_fwd_f16_v3_d64), reinterpret_cast<const void*>(g9_fmha_fwd_bf16_v3_d64)},
       {reinterpret_cast<const void*>(g9_fmha_fwd_f16_v4_d64), reinterpret_cast<const void*>(g9_fmha_fwd_bf16_v4_d64)}}};
  const void* fn = kFns[D == 64][variant == 4][dtype == G9_BF16];
  return hipLaunchKernel(fn, dim3((unsigned)(B * HQ * mblocks)), dim3(fa::kThreads), args, 0,
                         reinterpret_cast<hipStream_t>(stream)) == hipSuccess
             ? G9_OK
             : G9_ERR_HIP;
}

#ifdef G9_TIMING
#include "../../include/gfx950_gemm_timing.h"
extern "C" int g9_fmha_timing_read(void* host, size_t bytes) {
  if (bytes > sizeof(g9::fa::g9_fmha_timing_buf)) return G9_ERR_SHAPE;
  return hipMemcpyFromSymbol(host, HIP_SYMBOL(g9::fa::g9_fmha_timing_buf), bytes, 0, hipMemcpyDeviceToHost) ==
                 hipSuccess
             ? G9_OK
             : G9_ERR_HIP;
}
#endif
