// Rotary positions into packed rows (g9_rotary), and latents into a paged cache
// with their norm and rotation (g9_write_latent); declared in
// include/gfx950_fmha.h.
//
// A pair (a, b) at position n is turned by the angle n f: (a cos - b sin, a sin +
// b cos), in fp32 and rounded once.  The angle is formed in 64 bits: a product in 32
// would be off by whole radians where n f passes 2^24, and at position 10^5 by
// 2^-7.  f / 2 pi turns the product into whole turns, which are dropped exactly,
// and a rest of at most half a turn, which fp32 holds to 2^-26.
#include "../../include/gfx950_fmha.h"
#include "g9_attn_host.hpp"
#include "g9_common.hpp"
#include "g9_fmha_pipe.hpp"

using namespace g9;
using namespace g9::host;

namespace {

typedef float f32x2 __attribute__((ext_vector_type(2)));

// (cos, sin) of 2 pi n turns, times scale.
G9_DEV f32x2 turn(double n, double turns, float scale) {
  const double t = n * turns;
  const float r = (float)(t - __builtin_rint(t));
  float s, c;
  sincospif(2.f * r, &s, &c);
  return f32x2{c * scale, s * scale};
}
constexpr double kInvTwoPi = 0.15915494309189533577;

template <bool BF16>
G9_DEV void unpack8(u32x4 x, float (&y)[8]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const f32x2 v = fa::unpack2<BF16>(x[e]);
    y[2 * e] = v.x, y[2 * e + 1] = v.y;
  }
}
template <bool BF16>
G9_DEV u32x4 pack8(const float (&y)[8]) {
  return u32x4{fa::pack2<BF16>(y[0], y[1]), fa::pack2<BF16>(y[2], y[3]), fa::pack2<BF16>(y[4], y[5]),
               fa::pack2<BF16>(y[6], y[7])};
}

struct RotaryParams {
  const char* x;
  char* o;
  const long long* positions;
  const double* freqs;
  long long x_t, x_h, o_t, o_h;  // token / head strides, bytes
  long long units;               // T * groups * items
  float scale, sign;             // of the sine: -1 turns back
  int H, groups;                 // a thread takes every `groups`-th head
  int items, turned;             // a row's 16-value pieces that turn, then its 8-value pieces that do not
  int first, half;               // bytes: the turned part's begin, half its length
};

// A thread has one place within the rows: 16 values that turn (eight pairs), or 8
// that are copied.  Its angles serve every head of its token that it takes.  Bound by HBM:
// 16384 rows of 40 heads of 128 67 us (4.9 TB/s, the rate of a large copy); 64 rows 3.8.
template <bool BF16, bool INTERLEAVED>
G9_DEV void rotary(const RotaryParams& p) {
  for (long long u = (long long)blockIdx.x * 256 + threadIdx.x; u < p.units; u += (long long)gridDim.x * 256) {
    const long long rest = u / p.items;
    const int item = (int)(u - rest * p.items);
    const long long t = rest / p.groups;
    int h = (int)(rest - t * p.groups);
    const char* x = p.x + t * p.x_t;
    char* o = p.o + t * p.o_t;
    if (item >= p.turned) {
      int at = (item - p.turned) * 16;
      if (at >= p.first) at += 2 * p.half;
      for (; h < p.H; h += p.groups)
        *reinterpret_cast<u32x4*>(o + h * p.o_h + at) = *reinterpret_cast<const u32x4*>(x + h * p.x_h + at);
      continue;
    }
    f32x2 cs[8];
    const double n = (double)p.positions[t];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      cs[i] = turn(n, p.freqs[8 * item + i] * kInvTwoPi, p.scale);
      cs[i].y *= p.sign;
    }
    const int a_at = p.first + (INTERLEAVED ? 32 * item : 16 * item), b_at = a_at + (INTERLEAVED ? 16 : p.half);
    for (; h < p.H; h += p.groups) {
      float a[8], b[8];
      unpack8<BF16>(*reinterpret_cast<const u32x4*>(x + h * p.x_h + a_at), a);
      unpack8<BF16>(*reinterpret_cast<const u32x4*>(x + h * p.x_h + b_at), b);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        // Pair i: (a[i], b[i]), or neighbours of one of the two pieces.
        float& u0 = INTERLEAVED ? (i < 4 ? a[2 * i] : b[2 * i - 8]) : a[i];
        float& u1 = INTERLEAVED ? (i < 4 ? a[2 * i + 1] : b[2 * i - 7]) : b[i];
        const float v0 = u0 * cs[i].x - u1 * cs[i].y, v1 = u0 * cs[i].y + u1 * cs[i].x;
        u0 = v0, u1 = v1;
      }
      *reinterpret_cast<u32x4*>(o + h * p.o_h + a_at) = pack8<BF16>(a);
      *reinterpret_cast<u32x4*>(o + h * p.o_h + b_at) = pack8<BF16>(b);
    }
  }
}

struct LatentWriteParams {
  const char* c;
  const char* k;
  char* cache;
  char* c_out;  // or null
  char* k_out;  // or null
  const char* weight;  // or null: no norm
  const long long* slots;
  const long long* positions;
  const double* freqs;  // or null: no rotation
  long long c_t, k_t, co_t, ko_t;  // row strides, bytes
  long long b_b, b_t;              // cache block / token strides, bytes
  long long num_slots, T;
  float eps, scale;
  int shift;
};

// A wave per token: 8 of the latent's 512 values a lane, their squares' sum in fp32
// across the wave; of the 32 pairs of the key one a lane.  Bound by HBM: 16384 tokens, with
// c_out and k_out, 12.1-12.8 us (4.5 TB/s); 64 tokens 3.3.
template <bool BF16, bool INTERLEAVED>
G9_DEV void write_latent(const LatentWriteParams& p) {
  const int lane = threadIdx.x & 63;
  const long long waves = (long long)gridDim.x * 4;
  for (long long t = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); t < p.T; t += waves) {
    const long long slot = p.slots[t];
    u32x4 c = *reinterpret_cast<const u32x4*>(p.c + t * p.c_t + lane * 16);
    u32 pair = 0;
    const int pr = lane & 31;
    const char* const k = p.k + t * p.k_t;
    if constexpr (INTERLEAVED)
      pair = *reinterpret_cast<const u32*>(k + pr * 4);
    else
      pair = *reinterpret_cast<const uint16_t*>(k + pr * 2) | (u32)*reinterpret_cast<const uint16_t*>(k + 64 + pr * 2) << 16;
    if (p.weight) {
      float x[8], w[8];
      unpack8<BF16>(c, x);
      unpack8<BF16>(*reinterpret_cast<const u32x4*>(p.weight + lane * 16), w);
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum = __builtin_fmaf(x[i], x[i], sum);
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d, 64);
      const float r = 1.f / __builtin_sqrtf(sum * (1.f / 512) + p.eps);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = x[i] * r * w[i];
      c = pack8<BF16>(x);
    }
    if (p.freqs) {
      const f32x2 cs = turn((double)p.positions[t], p.freqs[pr] * kInvTwoPi, p.scale);
      const f32x2 v = fa::unpack2<BF16>(pair);
      pair = fa::pack2<BF16>(v.x * cs.x - v.y * cs.y, v.x * cs.y + v.y * cs.x);
    }
    const auto store_k = [&](char* to) {
      if (lane >= 32) return;
      if constexpr (INTERLEAVED) {
        *reinterpret_cast<u32*>(to + pr * 4) = pair;
      } else {
        *reinterpret_cast<uint16_t*>(to + pr * 2) = (uint16_t)pair;
        *reinterpret_cast<uint16_t*>(to + 64 + pr * 2) = (uint16_t)(pair >> 16);
      }
    };
    if (slot >= 0 && slot < p.num_slots) {
      char* const to = p.cache + (slot >> p.shift) * p.b_b + (slot & ((1ll << p.shift) - 1)) * p.b_t;
      *reinterpret_cast<u32x4*>(to + lane * 16) = c;
      store_k(to + 1024);
    }
    if (p.c_out) *reinterpret_cast<u32x4*>(p.c_out + t * p.co_t + lane * 16) = c;
    if (p.k_out) store_k(p.k_out + t * p.ko_t);
  }
}

#define G9_ROTARY_KERNELS(SUFFIX, BF16, INTERLEAVED)                                                                \
  extern "C" __global__ __launch_bounds__(256) void g9_rotary_##SUFFIX(RotaryParams p) {                            \
    rotary<BF16, INTERLEAVED>(p);                                                                                   \
  }                                                                                                                 \
  extern "C" __global__ __launch_bounds__(256) void g9_latent_write_##SUFFIX(LatentWriteParams p) {                 \
    write_latent<BF16, INTERLEAVED>(p);                                                                             \
  }
G9_ROTARY_KERNELS(f16_half, false, false)
G9_ROTARY_KERNELS(f16_pairs, false, true)
G9_ROTARY_KERNELS(bf16_half, true, false)
G9_ROTARY_KERNELS(bf16_pairs, true, true)
#define G9_ROTARY_FN(WHAT)                                                                               \
  {{reinterpret_cast<const void*>(WHAT##f16_half), reinterpret_cast<const void*>(WHAT##f16_pairs)},      \
   {reinterpret_cast<const void*>(WHAT##bf16_half), reinterpret_cast<const void*>(WHAT##bf16_pairs)}}
// [bf16][interleaved]
const void* const kRotary[2][2] = G9_ROTARY_FN(g9_rotary_);
const void* const kWrite[2][2] = G9_ROTARY_FN(g9_latent_write_);

bool finite(float x) { return (__builtin_bit_cast(uint32_t, x) >> 23 & 0xff) != 0xff; }

}  // namespace

extern "C" {

int g9_rotary(const void* x, void* o, const int64_t* positions, const double* freqs, int64_t T, int64_t H, int64_t D,
              int64_t first, int64_t dim, const int64_t* x_strides, const int64_t* o_strides, float scale,
              int interleaved, int inverse, int dtype, void* stream) {
  if (dtype != G9_F16 && dtype != G9_BF16) return G9_ERR_DTYPE;
  if (T < 0 || T > kMaxRows || H <= 0 || H > 65536 || D <= 0 || D > 65536 || D % 8 || first < 0 || first % 8 || dim <= 0 ||
      dim % 16 || first + dim > D || !finite(scale))
    return G9_ERR_SHAPE;
  if (!x_strides || !o_strides) return G9_ERR_LAYOUT;
  // The step of a single row is never taken.
  const int64_t xs[2] = {T > 1 ? x_strides[0] : 0, H > 1 ? x_strides[1] : 0};
  const int64_t os[2] = {T > 1 ? o_strides[0] : 0, H > 1 ? o_strides[1] : 0};
  if (!steps(xs, 2) || !steps(os, 2)) return G9_ERR_LAYOUT;
  const int64_t size[2] = {T, H};
  if (!apart(size, os, 2, D)) return G9_ERR_LAYOUT;
  if (T == 0) return G9_OK;
  if (!x || !o || !positions || !freqs) return G9_ERR_LAYOUT;
  if (!aligned16(x) || !aligned16(o) || ((uintptr_t)positions & 7) || ((uintptr_t)freqs & 7)) return G9_ERR_LAYOUT;
  const bool in_place = x == o && xs[0] == os[0] && xs[1] == os[1];
  if (x == o && !in_place) return G9_ERR_LAYOUT;
  RotaryParams p{};
  p.x = static_cast<const char*>(x);
  p.o = static_cast<char*>(o);
  p.positions = reinterpret_cast<const long long*>(positions);
  p.freqs = freqs;
  p.x_t = xs[0] * 2, p.x_h = xs[1] * 2, p.o_t = os[0] * 2, p.o_h = os[1] * 2;
  p.scale = scale;
  p.sign = inverse ? -1.f : 1.f;
  p.H = (int)H;
  p.turned = (int)(dim / 16);
  p.items = p.turned + (in_place ? 0 : (int)((D - dim) / 8));
  p.first = (int)(first * 2), p.half = (int)dim;
  const int64_t want = (256 * 2048 + T * p.items - 1) / (T * p.items);
  p.groups = (int)(want < H ? want : H);
  p.units = (long long)T * p.groups * p.items;
  const int64_t blocks = (p.units + 255) / 256;
  void* args[] = {&p};
  return launched(hipLaunchKernel(kRotary[dtype == G9_BF16][interleaved != 0],
                                  dim3((unsigned)(blocks < (1 << 23) ? blocks : 1 << 23)), dim3(256), args, 0,
                                  reinterpret_cast<hipStream_t>(stream)));
}

int g9_write_latent(const void* c, const void* k_rope, void* cache, const int64_t* slots, const void* weight, float eps,
                    const int64_t* positions, const double* freqs, void* c_out, void* k_out, int64_t T,
                    int64_t num_blocks, int64_t block_size, int64_t c_stride, int64_t k_stride,
                    const int64_t* cache_strides, int64_t c_out_stride, int64_t k_out_stride, float scale,
                    int interleaved, int dtype, void* stream) {
  if (dtype != G9_F16 && dtype != G9_BF16) return G9_ERR_DTYPE;
  if (T < 0 || T > kMaxRows || num_blocks < 0 || num_blocks > kMaxRows || !block_size_ok(block_size) || !finite(scale) ||
      !finite(eps) || eps < 0)
    return G9_ERR_SHAPE;
  if (!cache_strides || !steps(cache_strides, 2)) return G9_ERR_LAYOUT;
  const int64_t size[2] = {num_blocks, block_size};
  if (!apart(size, cache_strides, 2, 576)) return G9_ERR_LAYOUT;
  const int64_t in[2] = {T > 1 ? c_stride : 0, T > 1 ? k_stride : 0};
  const int64_t out[2] = {T > 1 && c_out ? c_out_stride : 512, T > 1 && k_out ? k_out_stride : 64};
  if (!steps(in, 2) || !steps(out, 2) || out[0] < 512 || out[1] < 64) return G9_ERR_LAYOUT;
  if (T == 0) return G9_OK;
  if (!c || !k_rope || !slots || (num_blocks && !cache) || (freqs && !positions)) return G9_ERR_LAYOUT;
  for (const void* q : {c, k_rope, (const void*)cache, weight, (const void*)c_out, (const void*)k_out})
    if (!aligned16(q)) return G9_ERR_LAYOUT;
  // In place a row's wave reads what it writes; with other steps it would write rows that are not read yet.
  if (T > 1 && ((c_out == c && out[0] != in[0]) || (k_out == k_rope && out[1] != in[1]))) return G9_ERR_LAYOUT;
  if (((uintptr_t)slots | (uintptr_t)positions | (uintptr_t)freqs) & 7) return G9_ERR_LAYOUT;
  LatentWriteParams p{};
  p.c = static_cast<const char*>(c);
  p.k = static_cast<const char*>(k_rope);
  p.cache = static_cast<char*>(cache);
  p.c_out = static_cast<char*>(c_out);
  p.k_out = static_cast<char*>(k_out);
  p.weight = static_cast<const char*>(weight);
  p.slots = reinterpret_cast<const long long*>(slots);
  p.positions = reinterpret_cast<const long long*>(positions);
  p.freqs = freqs;
  p.c_t = in[0] * 2, p.k_t = in[1] * 2, p.co_t = out[0] * 2, p.ko_t = out[1] * 2;
  p.b_b = cache_strides[0] * 2, p.b_t = cache_strides[1] * 2;
  p.num_slots = num_blocks * block_size;
  p.T = T;
  p.eps = eps, p.scale = scale;
  p.shift = log2_of(block_size);
  const int64_t blocks = (T + 3) / 4;
  void* args[] = {&p};
  return launched(hipLaunchKernel(kWrite[dtype == G9_BF16][interleaved != 0],
                                  dim3((unsigned)(blocks < (1 << 23) ? blocks : 1 << 23)), dim3(256), args, 0,
                                  reinterpret_cast<hipStream_t>(stream)));
}

}  // extern "C"
