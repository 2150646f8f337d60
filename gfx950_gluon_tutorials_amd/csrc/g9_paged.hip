// The paged cache's bookkeeping: block tables and slot maps, and rows into the
// cache (declared in include/gfx950_fmha.h).
#include "../../include/gfx950_fmha.h"
#include "g9_attn_host.hpp"
#include "g9_common.hpp"

using namespace g9;
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

extern "C" __global__ __launch_bounds__(kSlotThreads) void g9_slots(SlotParams p) {
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
  int tokens;                                      // of a wave
};

// A wave copies `tokens` tokens, one where a token's rows fill it: 16 bytes of K
// and of V per lane and step.  Bound by HBM: 16384 rows of 8 heads of 128 take
// 27.6 us, 4.9 TB/s, what a large copy reaches; 64 rows 2.6 us.
extern "C" __global__ __launch_bounds__(256) void g9_cache_write(WriteParams p) {
  const int n = p.HK << p.chunks_log2, sub = threadIdx.x & 63;
  const int in = p.tokens > 1 ? sub / n : 0, lane = sub - in * n;
  const long long wg = (long long)blockIdx.y * gridDim.x + blockIdx.x;
  const long long at = (wg * 4 + (threadIdx.x >> 6)) * p.tokens + in;
  if (at >= p.T || in >= p.tokens) return;
  const int t = (int)at;
  const long long slot = p.slots[t];
  if (slot < 0 || slot >= p.num_slots) return;
  const long long blk = slot >> p.shift, off = slot & ((1ll << p.shift) - 1);
  const char* k = p.k + t * p.k_t;
  const char* v = p.v + t * p.v_t;
  char* kc = p.kc + blk * p.kc_b + off * p.kc_t;
  char* vc = p.vc + blk * p.vc_b + off * p.vc_t;
  for (int i = lane; i < n; i += 64) {
    const long long h = i >> p.chunks_log2, c = (i & ((1 << p.chunks_log2) - 1)) * 16;
    const u32x4 x = *reinterpret_cast<const u32x4*>(k + h * p.k_h + c);
    const u32x4 y = *reinterpret_cast<const u32x4*>(v + h * p.v_h + c);
    *reinterpret_cast<u32x4*>(kc + h * p.kc_h + c) = x;
    *reinterpret_cast<u32x4*>(vc + h * p.vc_h + c) = y;
  }
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
  const int64_t chunks = HK * D / 8, per = chunks < 64 ? 64 / chunks : 1;
  p.tokens = (int)per;
  // A dimension of a launch has fewer than 2^32 threads.
  const int64_t wgs = (T + 4 * per - 1) / (4 * per), row = wgs < (1 << 22) ? wgs : 1 << 22;
  void* args[] = {&p};
  return launched(hipLaunchKernel(reinterpret_cast<const void*>(g9_cache_write),
                                  dim3((unsigned)row, (unsigned)((wgs + row - 1) / row)), dim3(256), args, 0,
                                  reinterpret_cast<hipStream_t>(stream)));
}

}  // extern "C"
