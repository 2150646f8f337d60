// Host-side argument checks shared by the packed and the paged attention entries.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/gfx950_fmha.h"

namespace g9 {
namespace host {

inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

inline int launched(hipError_t e) { return e == hipSuccess ? G9_OK : G9_ERR_HIP; }

// Strides in elements: 16-byte steps, none negative.
inline bool steps(const int64_t* s, int n) {
  for (int i = 0; i < n; ++i)
    if (s[i] < 0 || s[i] % 8 || s[i] > (int64_t(1) << 40)) return false;
  return true;
}
// Whether the rows of D elements at these steps are apart: what is written
// must not overlap.
inline bool apart(const int64_t* size, const int64_t* stride, int n, int64_t D) {
  int order[3] = {0, 1, 2};
  for (int i = 0; i < n; ++i)
    for (int j = i + 1; j < n; ++j)
      if (stride[order[j]] < stride[order[i]]) {
        const int x = order[i];
        order[i] = order[j], order[j] = x;
      }
  int64_t reach = D;  // elements that the inner dimensions span
  for (int i = 0; i < n; ++i) {
    const int d = order[i];
    if (size[d] <= 1) continue;
    if (stride[d] < reach) return false;
    reach += stride[d] * (size[d] - 1);
  }
  return true;
}
inline int log2_of(int64_t x) {
  int n = 0;
  while ((int64_t(1) << n) < x) ++n;
  return n;
}
inline bool block_size_ok(int64_t s) { return s >= 16 && s <= 1024 && (s & (s - 1)) == 0; }
// By the bits: some sources are compiled without NaN semantics.
inline bool scale_ok(float s) {
  const uint32_t b = __builtin_bit_cast(uint32_t, s);
  return (b >> 31) == 0 && b != 0 && ((b >> 23) & 0xff) != 0xff;
}
constexpr int64_t kMaxRows = 0x7fffffff - 4096;


}  // namespace host
}  // namespace g9
