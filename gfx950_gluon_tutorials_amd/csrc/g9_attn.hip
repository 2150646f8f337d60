// Attention over packed sequences and over a paged cache, and the cache's
// bookkeeping (declared in include/gfx950_fmha.h).
#include "../../include/gfx950_fmha.h"
#include "g9_attn.hpp"
#include "g9_attn_host.hpp"

using namespace g9;
using namespace g9::at;
using namespace g9::host;

namespace {

// --- block tables and slot maps ---------------------------------------------
//
// Token i of request b sits at position p = lengths[b] + i, in its block
// j = p / size.  Blocks j < have = ceil(lengths[b] / size) are in the table;
// the others are the next free ones, in the order of the requests: block j of
// request b is free_blocks[start + base[b] + j - have], base the exclusive sum
// of the requests' new blocks.
//
// Every workgroup sums the requests' counts and new blocks itself (8 bytes a
// request, from L2) and then takes 256 tokens: a launch for the sums alone
// would cost more than they do.
constexpr int kSlotThreads = 256;

struct SlotParams {
  const int* lengths;
  const int* counts;
  int* table;
  const int* free_blocks;
  const int* free_start;  // or null: 0
  int* cu;
  long long* slots;
  long long* positions;
  int* taken;
  long long table_stride;
  int B, width, num_free, size, T;
};

// Blocks that request b's table row gains.
G9_DEV int new_blocks(const SlotParams& p, long long len, long long n) {
  const long long have = (len + p.size - 1) / p.size, all = (len + n + p.size - 1) / p.size;
  const long long top = all < p.width ? all : p.width;
  return top > have ? (int)(top - have) : 0;
}
G9_DEV int saturated(long long x) { return x > 0x7fffffff ? 0x7fffffff : (int)x; }

__global__ __launch_bounds__(kSlotThreads) void g9_slots(SlotParams p) {
  extern __shared__ int sm[];  // token ends [B], first new block [B], wave sums
  int* const end = sm;
  int* const base = sm + p.B;
  long long* const part = reinterpret_cast<long long*>(sm + ((2 * p.B + 1) & ~1));
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  // Thread i sums requests [i run, (i + 1) run).
  const int run = (p.B + kSlotThreads - 1) / kSlotThreads;
  const int b0 = min(tid * run, p.B), b1 = min(b0 + run, p.B);
  long long tok = 0, blk = 0;
  for (int b = b0; b < b1; ++b) {
    const long long len = max(p.lengths[b], 0), n = max(p.counts[b], 0);
    tok += n;
    blk += new_blocks(p, len, n);
  }
  long long it = tok, ib = blk;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const long long t = __shfl_up(it, d, 64), k = __shfl_up(ib, d, 64);
    if (lane >= d) it += t, ib += k;
  }
  if (lane == 63) part[2 * wave] = it, part[2 * wave + 1] = ib;
  __syncthreads();
  it -= tok, ib -= blk;
  long long all = 0;
  for (int w = 0; w < kSlotThreads / 64; ++w) {
    if (w < wave) it += part[2 * w], ib += part[2 * w + 1];
    all += part[2 * w + 1];
  }
  for (int b = b0; b < b1; ++b) {
    const long long len = max(p.lengths[b], 0), n = max(p.counts[b], 0);
    base[b] = saturated(ib);
    it += n;
    ib += new_blocks(p, len, n);
    end[b] = saturated(it);
    if (blockIdx.x == 0) p.cu[b + 1] = end[b];
  }
  if (blockIdx.x == 0 && tid == 0) p.cu[0] = 0, p.taken[0] = saturated(all);
  __syncthreads();
  const int start = p.free_start ? max(p.free_start[0], 0) : 0;
  for (long long t = (long long)blockIdx.x * kSlotThreads + tid; t < p.T; t += (long long)gridDim.x * kSlotThreads) {
    int lo = 0, hi = p.B;
    while (lo < hi) {
      const int m = (lo + hi) >> 1;
      if (end[m] <= t)
        lo = m + 1;
      else
        hi = m;
    }
    long long slot = -1, pos = 0;
    if (lo < p.B) {
      const u32 len = max(p.lengths[lo], 0);
      const u32 at = len + (u32)(t - (lo ? end[lo - 1] : 0));
      const u32 have = (u32)(((long long)len + p.size - 1) / p.size), j = at / (u32)p.size, off = at - j * (u32)p.size;
      pos = at;
      int id = -1;
      if (j < (u32)p.width) {
        int* const entry = p.table + lo * p.table_stride + j;
        if (j < have) {
          id = *entry;
        } else {
          const long long f = (long long)start + base[lo] + (j - have);
          if (f < p.num_free) id = p.free_blocks[f];
          // A new block begins with a new token.
          if (off == 0) *entry = id;
        }
      }
      if (id >= 0) slot = (long long)id * p.size + off;
    }
    p.slots[t] = slot;
    p.positions[t] = pos;
  }
}

// --- rows into the cache ------------------------------------------------------

struct WriteParams {
  const char* k;
  const char* v;
  char* kc;
  char* vc;
  const long long* slots;
  long long k_t, k_h, v_t, v_h;                    // token / head strides, bytes
  long long kc_b, kc_t, kc_h, vc_b, vc_t, vc_h;    // block / token / head strides, bytes
  long long num_slots;
  int T, HK, shift, chunks_log2;                   // log2 of the block size, of a row's 16-byte pieces
};

// A wave copies one token: 16 bytes of K and of V per lane and step.
__global__ __launch_bounds__(256) void g9_cache_write(WriteParams p) {
  const int t = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (t >= p.T) return;
  const long long slot = p.slots[t];
  if (slot < 0 || slot >= p.num_slots) return;
  const long long blk = slot >> p.shift, off = slot & ((1ll << p.shift) - 1);
  const char* k = p.k + t * p.k_t;
  const char* v = p.v + t * p.v_t;
  char* kc = p.kc + blk * p.kc_b + off * p.kc_t;
  char* vc = p.vc + blk * p.vc_b + off * p.vc_t;
  const int n = p.HK << p.chunks_log2;
  for (int i = lane; i < n; i += 64) {
    const long long h = i >> p.chunks_log2, c = (i & ((1 << p.chunks_log2) - 1)) * 16;
    const u32x4 x = *reinterpret_cast<const u32x4*>(k + h * p.k_h + c);
    const u32x4 y = *reinterpret_cast<const u32x4*>(v + h * p.v_h + c);
    *reinterpret_cast<u32x4*>(kc + h * p.kc_h + c) = x;
    *reinterpret_cast<u32x4*>(vc + h * p.vc_h + c) = y;
  }
}

// --- attention, one wave per query row and head -------------------------------

struct AttnParams {
  const char* q;
  const char* k;
  const char* v;
  char* o;
  float* lse;                                      // [HQ][T], or null
  const int* cu_q;
  const int* cu_k;                                 // packed keys
  long long q_t, q_h, o_t, o_h;                    // token / head strides, bytes
  long long k_b, k_t, k_h, v_b, v_t, v_h;          // (block,) token, head strides, bytes
  const int* table;                                // paged keys
  const int* lengths;
  const unsigned long long* mask;
  long long table_stride, num_blocks;
  int width, shift, words;
  int B, T, TK, HQ, HK, causal;
  float scale_log2;
};

// One pass with a running maximum m and sum l (log2 units): 64 keys at a
// time, lane i scoring key i; then each lane sums its HD / 64 columns of P V
// over the keys that the row may read.  Keys that it may not read are never
// multiplied, whatever their rows hold.
template <bool BF16, int HD, bool PAGED>
__global__ __launch_bounds__(256) void g9_attn_rows(AttnParams p) {
  __shared__ float qs[4][HD];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const long long item = (long long)blockIdx.x * 4 + wave;
  const int t = (int)(item / p.HQ), h = (int)(item - (long long)t * p.HQ);
  if (t >= p.T) return;
  const int b = sequence_of(p.cu_q, p.B, t);
  if (b >= p.B) return;
  const Span sq = span_of(p.cu_q, b, p.T);
  const int i = t - sq.first;
  if (i < 0) return;
  const int hk = (int)((long long)h * p.HK / p.HQ);
  const char* kb = p.k + hk * p.k_h;
  const char* vb = p.v + hk * p.v_h;
  int keys, first = 0, context = 0;
  if constexpr (PAGED) {
    context = max(p.lengths[b], 0);
    keys = (int)min((long long)context + sq.rows, (long long)p.width << p.shift);
  } else {
    const Span sk = span_of(p.cu_k, b, p.TK);
    first = sk.first;
    keys = sk.rows;
    if (p.causal) keys = min(keys, max(i + 1 + sk.rows - sq.rows, 0));
  }
  const char* qrow = p.q + t * p.q_t + h * p.q_h;
  if (lane < HD / 2) {
    const f32x2 x = unpack2<BF16>(reinterpret_cast<const u32*>(qrow)[lane]);
    qs[wave][2 * lane] = x.x * p.scale_log2;
    qs[wave][2 * lane + 1] = x.y * p.scale_log2;
  }
  constexpr int kCols = HD / 64;
  float m = -__builtin_inff(), l = 0.f, acc[kCols] = {};
  for (int j0 = 0; j0 < keys; j0 += 64) {
    const int j = j0 + lane;
    bool reads = j < keys;
    long long ko = -1, vo = -1;  // the key's rows; -1: a page outside the cache, read as zeros
    if constexpr (PAGED) {
      if (reads && j >= context) {
        const int n = j - context;
        if (p.mask)
          reads = n < 64 * p.words && ((p.mask[(long long)t * p.words + n / 64] >> (n & 63)) & 1);
        else
          reads = n <= i;
      }
      if (reads) {
        const int page = p.table[b * p.table_stride + (j >> p.shift)];
        if (page >= 0 && page < p.num_blocks) {
          const int off = j & ((1 << p.shift) - 1);
          ko = page * p.k_b + off * p.k_t;
          vo = page * p.v_b + off * p.v_t;
        }
      }
    } else if (reads) {
      ko = (long long)(first + j) * p.k_t;
      vo = (long long)(first + j) * p.v_t;
    }
    float s = 0.f;
    if (ko >= 0) {
      const u32x4* row = reinterpret_cast<const u32x4*>(kb + ko);
      for (int c = 0; c < HD / 8; ++c) {
        const u32x4 w = row[c];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const f32x2 x = unpack2<BF16>(w[e]);
          s = __builtin_fmaf(x.x, qs[wave][8 * c + 2 * e], s);
          s = __builtin_fmaf(x.y, qs[wave][8 * c + 2 * e + 1], s);
        }
      }
    }
    if (!reads) s = -__builtin_inff();
    const float top = fmaxf(m, wave_max(s));
    const float base = top == -__builtin_inff() ? 0.f : top;
    const float alpha = __builtin_amdgcn_exp2f(m - base);
    const float pj = reads ? __builtin_amdgcn_exp2f(s - base) : 0.f;
    l = l * alpha + wave_sum(pj);
#pragma unroll
    for (int c = 0; c < kCols; ++c) acc[c] *= alpha;
    m = top;
    const unsigned long long who = __builtin_amdgcn_ballot_w64(reads);
    for (int n = 0; n < 64; ++n) {
      if (!((who >> n) & 1)) continue;
      const float w = __shfl(pj, n, 64);
      const long long off = __shfl(vo, n, 64);
      if (off < 0) continue;
      if constexpr (kCols == 2) {
        const f32x2 x = unpack2<BF16>(reinterpret_cast<const u32*>(vb + off)[lane]);
        acc[0] = __builtin_fmaf(w, x.x, acc[0]);
        acc[1] = __builtin_fmaf(w, x.y, acc[1]);
      } else {
        const u32 x = reinterpret_cast<const uint16_t*>(vb + off)[lane];
        acc[0] = __builtin_fmaf(w, unpack2<BF16>(x).x, acc[0]);
      }
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  char* orow = p.o + t * p.o_t + h * p.o_h;
  if constexpr (kCols == 2)
    reinterpret_cast<u32*>(orow)[lane] = pack2<BF16>(acc[0] * inv, acc[1] * inv);
  else
    reinterpret_cast<uint16_t*>(orow)[lane] = (uint16_t)pack2<BF16>(acc[0] * inv, 0.f);
  if (p.lse && lane == 0)
    p.lse[(long long)h * p.T + t] = l == 0.f ? -__builtin_inff() : (m + __builtin_log2f(l)) * kLn2;
}

const void* rows_kernel(int dtype, int64_t D) {
  if (dtype == G9_BF16)
    return D == 128 ? reinterpret_cast<const void*>(g9_attn_rows<true, 128, true>)
                    : reinterpret_cast<const void*>(g9_attn_rows<true, 64, true>);
  return D == 128 ? reinterpret_cast<const void*>(g9_attn_rows<false, 128, true>)
                  : reinterpret_cast<const void*>(g9_attn_rows<false, 64, true>);
}

}  // namespace

extern "C" {

int g9_assign_slots(const int32_t* lengths, const int32_t* counts, int64_t B, int32_t* block_table,
                    int64_t table_stride, int64_t width, const int32_t* free_blocks, int64_t num_free,
                    const int32_t* free_start, int64_t block_size, int64_t T, int32_t* cu_seqlens, int64_t* slots,
                    int64_t* positions, int32_t* taken, void* stream) {
  if (B < 0 || B > G9_SLOTS_MAX_REQUESTS || width < 0 || width > kMaxRows || num_free < 0 || num_free > kMaxRows ||
      T < 0 || T > kMaxRows || block_size < 1 || block_size > (1 << 20))
    return G9_ERR_SHAPE;
  if (!cu_seqlens || !taken || (B && (!lengths || !counts)) || (B && width && !block_table) ||
      (num_free && !free_blocks) || (T && (!slots || !positions)))
    return G9_ERR_LAYOUT;
  if (B > 1 && table_stride < width) return G9_ERR_LAYOUT;
  SlotParams p{};
  p.lengths = lengths;
  p.counts = counts;
  p.table = block_table;
  p.free_blocks = free_blocks;
  p.free_start = free_start;
  p.cu = cu_seqlens;
  p.slots = reinterpret_cast<long long*>(slots);
  p.positions = reinterpret_cast<long long*>(positions);
  p.taken = taken;
  p.table_stride = table_stride;
  p.B = (int)B;
  p.width = (int)width;
  p.num_free = (int)num_free;
  p.size = (int)block_size;
  p.T = (int)T;
  const int64_t want = (T + kSlotThreads - 1) / kSlotThreads;
  const unsigned grid = (unsigned)(want < 1 ? 1 : want < 1024 ? want : 1024);
  const size_t lds = (size_t)((2 * B + 1) & ~1) * 4 + 2 * (kSlotThreads / 64) * 8;
  void* args[] = {&p};
  return launched(hipLaunchKernel(reinterpret_cast<const void*>(g9_slots), dim3(grid), dim3(kSlotThreads), args, lds,
                                  reinterpret_cast<hipStream_t>(stream)));
}

int g9_write_cache(const void* k, const void* v, void* k_cache, void* v_cache, const int64_t* slots, int64_t T,
                   int64_t HK, int64_t D, int64_t num_blocks, int64_t block_size, const int64_t* k_strides,
                   const int64_t* v_strides, const int64_t* kc_strides, const int64_t* vc_strides, void* stream) {
  if (T < 0 || T > kMaxRows || HK <= 0 || HK > (1 << 20) || (D != 64 && D != 128) || num_blocks < 0 ||
      num_blocks > kMaxRows || !block_size_ok(block_size))
    return G9_ERR_SHAPE;
  if (!k_strides || !v_strides || !kc_strides || !vc_strides) return G9_ERR_LAYOUT;
  if (!steps(k_strides, 2) || !steps(v_strides, 2) || !steps(kc_strides, 3) || !steps(vc_strides, 3))
    return G9_ERR_LAYOUT;
  const int64_t size[3] = {num_blocks, block_size, HK};
  if (!apart(size, kc_strides, 3, D) || !apart(size, vc_strides, 3, D)) return G9_ERR_LAYOUT;
  if (T == 0 || num_blocks == 0) return G9_OK;
  if (!k || !v || !k_cache || !v_cache || !slots) return G9_ERR_LAYOUT;
  if (!aligned16(k) || !aligned16(v) || !aligned16(k_cache) || !aligned16(v_cache) || ((uintptr_t)slots & 7))
    return G9_ERR_LAYOUT;
  WriteParams p{};
  p.k = static_cast<const char*>(k);
  p.v = static_cast<const char*>(v);
  p.kc = static_cast<char*>(k_cache);
  p.vc = static_cast<char*>(v_cache);
  p.slots = reinterpret_cast<const long long*>(slots);
  p.k_t = k_strides[0] * 2, p.k_h = k_strides[1] * 2, p.v_t = v_strides[0] * 2, p.v_h = v_strides[1] * 2;
  p.kc_b = kc_strides[0] * 2, p.kc_t = kc_strides[1] * 2, p.kc_h = kc_strides[2] * 2;
  p.vc_b = vc_strides[0] * 2, p.vc_t = vc_strides[1] * 2, p.vc_h = vc_strides[2] * 2;
  p.num_slots = num_blocks * block_size;
  p.T = (int)T;
  p.HK = (int)HK;
  p.shift = log2_of(block_size);
  p.chunks_log2 = log2_of(D / 8);
  void* args[] = {&p};
  return launched(hipLaunchKernel(reinterpret_cast<const void*>(g9_cache_write), dim3((unsigned)((T + 3) / 4)),
                                  dim3(256), args, 0, reinterpret_cast<hipStream_t>(stream)));
}

int g9_tree_fwd(const void* q, const void* k_cache, const void* v_cache, void* o, float* lse,
                const int32_t* block_table, int64_t table_stride, int64_t width, const int32_t* lengths,
                const int32_t* cu_q, const int64_t* tree_mask, int64_t words, int64_t B, int64_t T, int64_t HQ,
                int64_t HK, int64_t D, int64_t num_blocks, int64_t block_size, const int64_t* q_strides,
                const int64_t* kc_strides, const int64_t* vc_strides, const int64_t* o_strides, float sm_scale,
                int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  if (dtype != G9_F16 && dtype != G9_BF16) return G9_ERR_DTYPE;
  if (B < 0 || B > kMaxRows || T < 0 || T > kMaxRows || HQ <= 0 || HQ > 65536 || HK <= 0 || HQ % HK ||
      (D != 64 && D != 128) || !scale_ok(sm_scale) || num_blocks < 0 || num_blocks > kMaxRows || width < 0 ||
      width > kMaxRows || !block_size_ok(block_size) || width * block_size > kMaxRows || words < 0 || words > 1024 ||
      (tree_mask && words == 0))
    return G9_ERR_SHAPE;
  if (!q_strides || !kc_strides || !vc_strides || !o_strides) return G9_ERR_LAYOUT;
  if (!steps(q_strides, 2) || !steps(kc_strides, 3) || !steps(vc_strides, 3) || !steps(o_strides, 2))
    return G9_ERR_LAYOUT;
  const int64_t size[2] = {T, HQ};
  if (!apart(size, o_strides, 2, D) || (B > 1 && table_stride < width)) return G9_ERR_LAYOUT;
  if (B == 0 || T == 0) return G9_OK;
  if (!q || !o || !lengths || !cu_q || (width && !block_table) || (num_blocks && (!k_cache || !v_cache)))
    return G9_ERR_LAYOUT;
  if (!aligned16(q) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(o) || ((uintptr_t)lse & 3) ||
      ((uintptr_t)tree_mask & 7))
    return G9_ERR_LAYOUT;
  (void)workspace, (void)workspace_bytes;
  AttnParams p{};
  p.q = static_cast<const char*>(q);
  p.k = static_cast<const char*>(k_cache);
  p.v = static_cast<const char*>(v_cache);
  p.o = static_cast<char*>(o);
  p.lse = lse;
  p.cu_q = cu_q;
  p.q_t = q_strides[0] * 2, p.q_h = q_strides[1] * 2, p.o_t = o_strides[0] * 2, p.o_h = o_strides[1] * 2;
  p.k_b = kc_strides[0] * 2, p.k_t = kc_strides[1] * 2, p.k_h = kc_strides[2] * 2;
  p.v_b = vc_strides[0] * 2, p.v_t = vc_strides[1] * 2, p.v_h = vc_strides[2] * 2;
  p.table = block_table;
  p.table_stride = table_stride;
  p.lengths = lengths;
  p.mask = reinterpret_cast<const unsigned long long*>(tree_mask);
  p.words = (int)words;
  p.width = (int)width;
  p.num_blocks = num_blocks;
  p.shift = log2_of(block_size);
  p.B = (int)B, p.T = (int)T, p.HQ = (int)HQ, p.HK = (int)HK;
  p.causal = 1;
  p.scale_log2 = sm_scale * kLog2e;
  const int64_t waves = T * HQ;
  if ((waves + 3) / 4 > INT32_MAX) return G9_ERR_SHAPE;
  void* args[] = {&p};
  return launched(hipLaunchKernel(rows_kernel(dtype, D), dim3((unsigned)((waves + 3) / 4)), dim3(256), args, 0,
                                  reinterpret_cast<hipStream_t>(stream)));
}

size_t g9_tree_workspace_size(int64_t B, int64_t T, int64_t HQ, int64_t HK, int64_t D) {
  (void)B, (void)T, (void)HQ, (void)HK, (void)D;
  return 0;
}

}  // extern "C"
