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
#include "g9_fmha_pipe.hpp"

namespace g9 {
namespace fa {

struct VarParams {
  const char* q;
  const char* k;
  const char* v;
  char* o;
  float* lse;                                  // [HQ][T] fp32, or null
  const int* cu_q;
  const int* cu_k;
  long long q_h, k_h, v_h, o_h;                // head strides, bytes
  u32 ldq, ldk, ldv, ldo;                      // token strides, bytes
  int B, T, TK, HQ, HK, causal;
  float scale_log2;
};

struct Tile {
  int q0, lq, k0, lk, mb;  // the sequence's first query, queries, first key, keys; the tile
};

// Sum over the wave's lanes, in every lane.
G9_DEV int wave_add(int x) {
#pragma unroll
  for (int d = 32; d; d >>= 1) x += __shfl_xor(x, d, 64);
  return x;
}

// Sequence b's tiles: `n` of them, the last of cost `top` (in units of 256
// keys), the others one less each.
struct Cost {
  int n, top;
};
G9_DEV Cost cost_of(const VarParams& p, int b) {
  if (b >= p.B) return {0, 0};
  const int q0 = min(max(p.cu_q[b], 0), p.T), lq = min(max(p.cu_q[b + 1], q0), p.T) - q0;
  const int k0 = min(max(p.cu_k[b], 0), p.TK), lk = min(max(p.cu_k[b + 1], k0), p.TK) - k0;
  const int n = (lq + kBlockM - 1) / kBlockM;
  const int before = p.causal ? max(lk - lq, 0) : lk;
  return {n, n + (before + kBlockM - 1) / kBlockM};
}
// Tiles of a sequence that cost at least c; whether one costs exactly c.
G9_DEV int at_least(Cost s, int c) { return min(s.n, max(s.top - c + 1, 0)); }
G9_DEV bool exactly(Cost s, int c) { return c <= s.top && c > s.top - s.n; }

// Tile `rank` of the batch in the order of falling cost (equal costs in the
// order of the sequences).  C(c), the number of tiles that cost at least c,
// falls with c: the tile's cost is the largest c with C(c) > rank, found by
// bisection.  Batches of up to 64 sequences stay within a wave (a lane each);
// larger ones sum over the workgroup.  Returns false behind the last tile.
G9_DEV bool find_tile(const VarParams& p, int rank, int* lds, Tile& t) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int seq = -1, cost = 0;
  if (p.B <= 64) {
    const Cost s = cost_of(p, lane);
    if (rank >= wave_add(s.n)) return false;
    int hi = s.n ? s.top : 0;  // C(hi + 1) = 0 <= rank
#pragma unroll
    for (int d = 32; d; d >>= 1) hi = max(hi, __shfl_xor(hi, d, 64));
    int lo = 1;  // C(1) is all of them: every tile costs at least 1
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (wave_add(at_least(s, mid)) > rank)
        lo = mid;
      else
        hi = mid - 1;
    }
    cost = lo;
    const int nth = rank - wave_add(at_least(s, cost + 1));
    unsigned long long who = __builtin_amdgcn_ballot_w64(exactly(s, cost));
    for (int i = 0; i < nth; ++i) who &= who - 1;
    seq = __builtin_ctzll(who);
  } else {
    // Thread i holds the sequences i, i + 512, ... (again from memory each time:
    // they are in L1).
    const auto total = [&](auto f) {
      int x = 0;
      for (int b = tid; b < p.B; b += kThreads) x += f(cost_of(p, b));
      x = wave_add(x);
      __syncthreads();
      if (lane == 0) lds[wave] = x;
      __syncthreads();
      int all = 0;
      for (int w = 0; w < kWaves; ++w) all += lds[w];
      return all;
    };
    if (rank >= total([](Cost s) { return s.n; })) return false;
    // Keys and queries both fit 2^31: no tile costs more than 2^24.
    int lo = 1, hi = 1;
    while (total([&](Cost s) { return at_least(s, 2 * hi); }) > rank) lo = hi *= 2;
    hi = 2 * hi - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (total([&](Cost s) { return at_least(s, mid); }) > rank)
        lo = mid;
      else
        hi = mid - 1;
    }
    cost = lo;
    const int nth = rank - total([&](Cost s) { return at_least(s, cost + 1); });
    // The nth thread-major sequence of that cost.
    int mine = 0;
    for (int b = tid; b < p.B; b += kThreads) mine += exactly(cost_of(p, b), cost);
    int before = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int x = __shfl_up(before, d, 64);
      if (lane >= d) before += x;
    }
    __syncthreads();
    if (lane == 63) lds[wave] = before;
    __syncthreads();
    before -= mine;
    for (int w = 0; w < wave; ++w) before += lds[w];
    if (nth >= before && nth < before + mine) {
      int i = before;
      for (int b = tid; b < p.B; b += kThreads)
        if (exactly(cost_of(p, b), cost) && i++ == nth) lds[kWaves] = b;
    }
    __syncthreads();
    seq = lds[kWaves];
    __syncthreads();
  }
  seq = __builtin_amdgcn_readfirstlane(seq);
  cost = __builtin_amdgcn_readfirstlane(cost);
  const Cost s = cost_of(p, seq);
  t.mb = s.n - 1 - (s.top - cost);
  t.q0 = min(max(p.cu_q[seq], 0), p.T);
  t.lq = min(max(p.cu_q[seq + 1], t.q0), p.T) - t.q0;
  t.k0 = min(max(p.cu_k[seq], 0), p.TK);
  t.lk = min(max(p.cu_k[seq + 1], t.k0), p.TK) - t.k0;
  for (int* x : {&t.mb, &t.q0, &t.lq, &t.k0, &t.lk}) *x = __builtin_amdgcn_readfirstlane(*x);
  return true;
}

template <bool BF16, int HD>
struct VarPipe {
  using T = Pipe<VarParams, BF16, true, false, HD, kPacked>;
  static constexpr int kLds = T::kLdsBytes + kWaves * T::kScratchBytes;
};

template <bool BF16, int HD>
G9_DEV void varlen_fwd(const VarParams& p, char* smem) {
  using PipeT = typename VarPipe<BF16, HD>::T;
  // Workgroups go round the 8 XCDs.  (tile rank, K/V head) pairs are dealt to
  // the XCDs in turn and the query heads of a pair stay together, so that what
  // runs on an XCD at a time reads few K/V heads from its L2; with a multiple of
  // 8 K/V heads each keeps to one XCD.
  const int group = p.HQ / p.HK;
  const int turn = blockIdx.x >> 3;
  const int pair = 8 * (turn / group) + (int)(blockIdx.x & 7);
  const int rank = pair / p.HK, hk = pair - rank * p.HK;
  const int hq = hk * group + turn % group;
  Tile t;
  if (!find_tile(p, rank, reinterpret_cast<int*>(smem), t)) return;

  const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5;
  PipeT P(p);
  P.wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wave = P.wave;
  // Query i reads the keys below i + 1 + shift.
  const int shift = p.causal ? t.lk - t.lq : t.lk;
  const auto limit = [&](int i) { return min(max(min(i, t.lq - 1) + 1 + shift, 0), t.lk); };
  const int last = min((t.mb + 1) * kBlockM, t.lq) - 1;
  const int qrow = t.mb * kBlockM + wave * 32 + (lane & 31);
  P.keys = t.lk;
  P.lim = limit(qrow);
  P.wlim = limit(t.mb * kBlockM + wave * 32);
  P.nt = (limit(last) + PipeT::kBN - 1) / PipeT::kBN;
  P.nte = max((P.nt + 1) & ~1, 2);
  P.lds0 = (u32)(uintptr_t)to_lds(smem);
  P.pscratch = smem + PipeT::kLdsBytes + wave * PipeT::kScratchBytes;
  const int nte = P.nte;
  const char* qb = p.q + hq * p.q_h + (size_t)(t.q0 + t.mb * kBlockM) * p.ldq;
  const rsrc_t rq = make_rsrc(qb, (u32)min(t.lq - t.mb * kBlockM, kBlockM) * p.ldq);
  P.kp = p.k + hk * p.k_h + (size_t)t.k0 * p.ldk;
  P.vp = p.v + hk * p.v_h + (size_t)t.k0 * p.ldv;
#pragma unroll
  for (int s = 0; s < PipeT::kNS; ++s)
    P.qf[s] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                            rq, (u32)(wave * 32 + (lane & 31)) * p.ldq + (16 * s + 8 * h) * 2, 0, 0));
  P.voffk = (u32)lane * p.ldk;
  P.voffv = (u32)lane * p.ldv;
  P.ak = P.lds0 + h * PipeT::kPitchK + (lane & 31) * 16;
  {
    const int G = lane >> 4, jj = lane & 15;
    P.av = P.lds0 + PipeT::kLdsV + (2 * (G & 1) + ((jj & 3) >> 1)) * PipeT::kPitchV + (4 * (G >> 1) + (jj >> 2)) * 16 +
           8 * (jj & 1);
  }
  // The prologue of the equal-length kernel: K_0, V_0, K_1 in; S_0 and its first
  // softmax half; K_2 and V_1 requested; K_1 in registers.
  P.dma_k(0, 0);
  P.dma_v(0, 0);
  P.dma_k(1, 1);
  P.sc = p.scale_log2;
#pragma unroll
  for (int d = 0; d < PipeT::kND; ++d) P.o[d] = f32x16{};
  // Finite, so that a row whose keys so far are all masked has weights
  // 2^(-inf - m) = 0 and a sum of 0, not NaN.
  P.m = -3.0e38f;
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
  if (P.masked(0)) P.mask_tile(sa, 0);
  P.vec0(sa);
  P.vec1(sa);
  P.l *= P.alpha;
  P.template read_k<1>();
  waitcnt<63, 0>();

  const bool lag = wave >= 4;
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

  const float lt = xhalf(P.l, [](float x, float y) { return x + y; });
  // By its bits: comparisons here may take NaN for a number.
  const bool none = (__float_as_uint(lt) << 1) == 0;
  const float inv = none ? 0.f : 1.f / lt;
  if (qrow < t.lq) {
    char* orow = p.o + hq * p.o_h + (size_t)(t.q0 + qrow) * p.ldo;
#pragma unroll
    for (int d = 0; d < PipeT::kND; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int col = 32 * d + 8 * r + 4 * h;
        const u32x2 w = {pack2<BF16>(P.o[d][4 * r] * inv, P.o[d][4 * r + 1] * inv),
                         pack2<BF16>(P.o[d][4 * r + 2] * inv, P.o[d][4 * r + 3] * inv)};
        *reinterpret_cast<u32x2*>(orow + col * 2) = w;
      }
    if (p.lse && h == 0)
      p.lse[(size_t)hq * p.T + t.q0 + qrow] =
          none ? -__builtin_inff() : (P.m + __builtin_log2f(lt)) * kLn2;
  }
}

}  // namespace fa
}  // namespace g9

using namespace g9;
using namespace g9::host;

#define G9_VARLEN_KERNEL(NAME, BF16, HD)                                                                   \
  extern "C" __global__ __launch_bounds__(fa::kThreads) __attribute__((amdgpu_waves_per_eu(2, 2))) void \
  NAME(fa::VarParams p) {                                                                                 \
    __shared__ __attribute__((aligned(1024))) char smem[fa::VarPipe<BF16, HD>::kLds];                      \
    fa::varlen_fwd<BF16, HD>(p, smem);                                                                    \
  }
G9_VARLEN_KERNEL(g9_varlen_bf16, true, 128)
G9_VARLEN_KERNEL(g9_varlen_f16, false, 128)
G9_VARLEN_KERNEL(g9_varlen_bf16_d64, true, 64)
G9_VARLEN_KERNEL(g9_varlen_f16_d64, false, 64)

extern "C" int g9_varlen_fwd(const void* q, const void* k, const void* v, void* o, float* lse, const int32_t* cu_q,
                  const int32_t* cu_k, int64_t B, int64_t T, int64_t TK, int64_t HQ, int64_t HK, int64_t D,
                  const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides,
                  const int64_t* o_strides, float sm_scale, int dtype, int causal, void* stream) {
  if (dtype != G9_F16 && dtype != G9_BF16) return G9_ERR_DTYPE;
  if (B < 0 || B > kMaxRows || T < 0 || T > kMaxRows || TK < 0 || TK > kMaxRows || HQ <= 0 || HQ > 65536 || HK <= 0 ||
      HQ % HK || (D != 64 && D != 128) || !scale_ok(sm_scale))
    return G9_ERR_SHAPE;
  if (!q_strides || !k_strides || !v_strides || !o_strides) return G9_ERR_LAYOUT;
  if (!steps(q_strides, 2) || !steps(k_strides, 2) || !steps(v_strides, 2) || !steps(o_strides, 2))
    return G9_ERR_LAYOUT;
  const int64_t size[2] = {T, HQ};
  if (!apart(size, o_strides, 2, D)) return G9_ERR_LAYOUT;
  if (B == 0 || T == 0) return G9_OK;
  if (!q || !o || (TK && (!k || !v)) || !cu_q || !cu_k) return G9_ERR_LAYOUT;
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(o) || ((uintptr_t)lse & 3)) return G9_ERR_LAYOUT;
  // Token strides within 32 bits, a tile's rows within a descriptor's range.
  for (const int64_t* st : {q_strides, k_strides, v_strides, o_strides})
    if (st[0] * 2 * fa::kBlockM >= (int64_t(1) << 31)) return G9_ERR_LAYOUT;
  fa::VarParams p{};
  p.q = static_cast<const char*>(q);
  p.k = static_cast<const char*>(k);
  p.v = static_cast<const char*>(v);
  p.o = static_cast<char*>(o);
  p.lse = lse;
  p.cu_q = cu_q;
  p.cu_k = cu_k;
  p.q_h = q_strides[1] * 2, p.k_h = k_strides[1] * 2, p.v_h = v_strides[1] * 2, p.o_h = o_strides[1] * 2;
  p.ldq = (u32)(q_strides[0] * 2), p.ldk = (u32)(k_strides[0] * 2);
  p.ldv = (u32)(v_strides[0] * 2), p.ldo = (u32)(o_strides[0] * 2);
  p.B = (int)B, p.T = (int)T, p.TK = (int)TK, p.HQ = (int)HQ, p.HK = (int)HK;
  p.causal = causal != 0;
  p.scale_log2 = sm_scale * fa::kLog2e;
  // At most T / 256 whole tiles and a partial one per sequence.
  const int64_t tiles = T / fa::kBlockM + (B < T ? B : T);
  const int64_t grid = 8 * (HQ / HK) * ((tiles * HK + 7) / 8);
  if (grid > INT32_MAX) return G9_ERR_SHAPE;
  static const void* const kFns[2][2] = {
      {reinterpret_cast<const void*>(g9_varlen_f16), reinterpret_cast<const void*>(g9_varlen_bf16)},
      {reinterpret_cast<const void*>(g9_varlen_f16_d64), reinterpret_cast<const void*>(g9_varlen_bf16_d64)}};
  void* args[] = {&p};
  return launched(hipLaunchKernel(kFns[D == 64][dtype == G9_BF16], dim3((unsigned)grid), dim3(fa::kThreads), args, 0,
                                  reinterpret_cast<hipStream_t>(stream)));
}
