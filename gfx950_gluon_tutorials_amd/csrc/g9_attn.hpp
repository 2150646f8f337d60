// Shared by the packed and the paged attention kernels: 16-bit element
// conversions, wave reductions and the lookup of a packed row's sequence.
#pragma once

#include <stdint.h>

#include "g9_common.hpp"

namespace g9 {
namespace at {

typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// Two 16-bit values of one register -> fp32.
template <bool BF16>
G9_DEV f32x2 unpack2(u32 w) {
  if constexpr (BF16) {
    return f32x2{__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)};
  } else {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    return __builtin_convertvector(__builtin_bit_cast(h2, w), f32x2);
  }
}
// Two fp32 values -> one register of two 16-bit values (round to nearest even).
template <bool BF16>
G9_DEV u32 pack2(float x, float y) {
  if constexpr (BF16) {
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(u32, __builtin_convertvector((f32x2){x, y}, b2));
  } else {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(u32, __builtin_convertvector((f32x2){x, y}, h2));
  }
}

G9_DEV float wave_max(float x) {
#pragma unroll
  for (int d = 32; d; d >>= 1) x = fmaxf(x, __shfl_xor(x, d, 64));
  return x;
}
G9_DEV float wave_sum(float x) {
#pragma unroll
  for (int d = 32; d; d >>= 1) x += __shfl_xor(x, d, 64);
  return x;
}

// Rows [first, first + rows) of sequence b in a packed tensor of T rows; the
// offsets are device data, so they are held inside the tensor here.
struct Span {
  int first, rows;
};
G9_DEV Span span_of(const int* cu, int b, int T) {
  const int a = min(max(cu[b], 0), T), e = min(max(cu[b + 1], a), T);
  return {a, e - a};
}
// The sequence of packed row t: the number of sequence ends at or before t (B
// for a row behind the last sequence).
G9_DEV int sequence_of(const int* cu, int B, int t) {
  int lo = 0, hi = B;
  while (lo < hi) {
    const int m = (lo + hi) >> 1;
    if (cu[m + 1] <= t)
      lo = m + 1;
    else
      hi = m;
  }
  return lo;
}

}  // namespace at
}  // namespace g9
