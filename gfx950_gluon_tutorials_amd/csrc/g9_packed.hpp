// Attention over packed sequences on the pipeline of g9_fmha_pipe.hpp
// (g9_varlen.hip, g9_latent_varlen.hip): which tile of which sequence a workgroup
// takes, and its walk over the keys.
#pragma once

#include "g9_wave.hpp"

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

  // A query row of the short form: its place, the keys before the sequence's
  // first query (all of them without a mask).
  struct Row {
    int node, context, q0;
  };
  // Bit i: the row reads key k0 + i of `keys`.
  G9_DEV unsigned long long reads(const Row& r, int k0, int keys) const {
    const int c = min(r.node + 1 + r.context, keys) - k0;
    return c >= 64 ? ~0ull : c <= 0 ? 0 : (1ull << c) - 1;
  }
};

struct Tile {
  int q0, lq, k0, lk, mb;  // the sequence's first query, queries, first key, keys; the tile
};

// Sum over the wave's lanes: rows of 16, then across them (the DPP moves take a
// few cycles each where a shuffle goes through LDS).
G9_DEV int wave_add(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr 1, 2, 4, 8
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast 15
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast 31
  return __builtin_amdgcn_readlane(x, 63);
}

// Sequence b's tiles of BLOCK rows, `per` rows a query: `n` of them, the last of
// cost `top` (in units of BLOCK / per keys), the others one less each.
struct Cost {
  int n, top;
};
template <int BLOCK, class P>
G9_DEV Cost cost_of(const P& p, int b, int per) {
  if (b >= p.B) return {0, 0};
  const int q0 = min(max(p.cu_q[b], 0), p.T), lq = min(max(p.cu_q[b + 1], q0), p.T) - q0;
  const int k0 = min(max(p.cu_k[b], 0), p.TK), lk = min(max(p.cu_k[b + 1], k0), p.TK) - k0;
  const auto blocks = [&](int x) { return (int)min(((long long)x * per + BLOCK - 1) / BLOCK, 1ll << 28); };
  const int n = blocks(lq);
  return {n, n + blocks(p.causal ? max(lk - lq, 0) : lk)};
}
// Tiles of a sequence that cost at least c; whether one costs exactly c.
G9_DEV int at_least(Cost s, int c) { return min(s.n, max(s.top - c + 1, 0)); }
G9_DEV bool exactly(Cost s, int c) { return c <= s.top && c > s.top - s.n; }

// Tile `rank` of the batch in the order of falling cost (equal costs in the
// order of the sequences).  C(c), the number of tiles that cost at least c,
// falls with c: the tile's cost is the largest c with C(c) > rank, found by
// bisection.  Batches of up to 64 sequences stay within a wave (a lane each);
// larger ones sum over the workgroup.  Returns false behind the last tile.
template <int BLOCK, int THREADS, class P>
G9_DEV bool find_tile(const P& p, int rank, int per, int* lds, Tile& t) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int seq = -1, cost = 0;
  if (p.B == 1) {
    const Cost s = cost_of<BLOCK>(p, 0, per);
    if (rank >= s.n) return false;
    seq = 0, cost = s.top - rank;
  } else if (p.B <= 64) {
    const Cost s = cost_of<BLOCK>(p, lane, per);
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
    // Thread i holds the sequences i, i + THREADS, ... (again from memory each time:
    // they are in L1).
    const auto total = [&](auto f) {
      int x = 0;
      for (int b = tid; b < p.B; b += THREADS) x += f(cost_of<BLOCK>(p, b, per));
      x = wave_add(x);
      __syncthreads();
      if (lane == 0) lds[wave] = x;
      __syncthreads();
      int all = 0;
      for (int w = 0; w < (THREADS / 64); ++w) all += lds[w];
      return all;
    };
    if (rank >= total([](Cost s) { return s.n; })) return false;
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
    for (int b = tid; b < p.B; b += THREADS) mine += exactly(cost_of<BLOCK>(p, b, per), cost);
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
      for (int b = tid; b < p.B; b += THREADS)
        if (exactly(cost_of<BLOCK>(p, b, per), cost) && i++ == nth) lds[(THREADS / 64)] = b;
    }
    __syncthreads();
    seq = lds[(THREADS / 64)];
    __syncthreads();
  }
  // Held inside whatever the offsets say (sums of more than 2^31 tiles wrap).
  seq = min(max(__builtin_amdgcn_readfirstlane(seq), 0), p.B - 1);
  cost = __builtin_amdgcn_readfirstlane(cost);
  const Cost s = cost_of<BLOCK>(p, seq, per);
  t.mb = s.n - 1 - (s.top - cost);
  t.q0 = min(max(p.cu_q[seq], 0), p.T);
  t.lq = min(max(p.cu_q[seq + 1], t.q0), p.T) - t.q0;
  t.k0 = min(max(p.cu_k[seq], 0), p.TK);
  t.lk = min(max(p.cu_k[seq + 1], t.k0), p.TK) - t.k0;
  for (int* x : {&t.mb, &t.q0, &t.lq, &t.k0, &t.lk}) *x = __builtin_amdgcn_readfirstlane(*x);
  return (u32)t.mb < (u32)s.n;
}

template <class P, bool BF16, int HD, int ROPE = 0>
struct VarPipe {
  using T = Pipe<P, BF16, true, false, HD, kPacked, ROPE>;
  static constexpr int kLds = T::kLdsBytes + kWaves * T::kScratchBytes;
};

template <bool BF16, int HD, int ROPE = 0, class Params>
G9_DEV void varlen_fwd(const Params& p, char* smem) {
  using PipeT = typename VarPipe<Params, BF16, HD, ROPE>::T;
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
  if (!find_tile<kBlockM, kThreads>(p, rank, 1, reinterpret_cast<int*>(smem), t)) return;

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
  const rsrc_t rq = make_rsrc(qb, extent(min(t.lq - t.mb * kBlockM, kBlockM), p.ldq, (HD + ROPE) * 2));
  P.kp = p.k + hk * p.k_h + (size_t)t.k0 * p.ldk;
  P.vp = p.v + hk * p.v_h + (size_t)t.k0 * p.ldv;
#pragma unroll
  for (int s = 0; s < PipeT::kNS + PipeT::kNR; ++s)
    P.qf[s] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                            rq, (u32)(wave * 32 + (lane & 31)) * p.ldq + (16 * s + 8 * h) * 2, 0, 0));
  if constexpr (ROPE != 0) {
    P.rp = p.r + (size_t)t.k0 * p.ldr;
    P.voffr = (u32)lane * p.ldr;
  }
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
  P.dma_r(0, 0);
  P.dma_v(0, 0);
  P.dma_k(1, 1);
  P.dma_r(1, 1);
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
  if (nte > 2) {
    P.dma_k(2, 0);
    P.dma_r(2, 0);
  }
  P.dma_v(1, 1);
  if (P.masked(0)) P.mask_tile(sa, 0);
  P.vec0(sa);
  P.vec1(sa);
  P.l *= P.alpha;
  P.template read_k<1>();
  waitcnt<63, 0>();

  const bool lag = wave >= 4;
  if (lag) barrier();
  // The tiles that a row of this wave reads, rounded up to even; the others are
  // left to the waves behind it (a quarter of a 256-query prompt's tiles, and most of
  // a short last block's).
  const int w0 = t.mb * kBlockM + wave * 32;
  const int own = w0 < t.lq ? min(max(((limit(w0 + 31) + PipeT::kBN - 1) / PipeT::kBN + 1) & ~1, 2), nte) : 2;
  int j = 0;
  for (; j + 2 < own; j += 2) {
    P.template step<0, true>(j, sa, sb);
    P.template step<1, true>(j + 1, sb, sa);
  }
  P.template step<0, true>(j, sa, sb);
  P.template step<1, false>(j + 1, sb, sa);
  __builtin_amdgcn_s_setprio(0);
  for (j += 2; j < nte; ++j) P.idle(j);
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

// Few queries: a workgroup per 32 rows (queries by the query heads of a K/V head),
// its 4 waves taking the key tiles in turn and joining their sums in LDS; two
// workgroups a CU, so that one computes while the other waits for its tile (one,
// with two stages a wave: 66 us for 2048 queries instead of 38).  The pipeline's
// workgroups of 256 queries leave most of the chip idle there, and its 60 KB of code
// are fetched for a few tiles.
template <class P, bool BF16, int HD, int ROPE = 0>
struct ShortWave {
  using T = Wave<P, BF16, HD, 1, 1, ROPE>;
  static constexpr int kLds = 4 * T::kWaveLds;
};
template <bool BF16, int HD, int ROPE = 0, class Params>
G9_DEV void varlen_short(const Params& p, char* smem) {
  using W = typename ShortWave<Params, BF16, HD, ROPE>::T;
  const int group = p.HQ / p.HK;
  const int rank = blockIdx.x / p.HK, hk = blockIdx.x - rank * p.HK;
  Tile t;
  if (!find_tile<32, 256>(p, rank, group, reinterpret_cast<int*>(smem), t)) return;
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  W w(p);
  w.init(smem, wave, p.ldk, p.ldv);
  if constexpr (ROPE != 0) w.init_shared(p.ldr);
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
      if constexpr (ROPE != 0)
        w.fill_shared(i, p.r + (size_t)(u32)(t.k0 + k) * p.ldr, min(max(t.lk - k, 0), 16), p.ldr);
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
