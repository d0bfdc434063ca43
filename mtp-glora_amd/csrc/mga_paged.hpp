// Shared by the kernels of the paged 8-bit cache: its layout, and which tokens
// belong to which sequence.
//
// A page holds PS (16, 32, 64 or 128) tokens of every head. Keys lie [page, head,
// row, channel], values [page, head, channel, row], one e4m3 byte each: both are
// then read by the attention as its matrix instructions take them, 16 bytes a lane
// along the products' inner dimension, with no transpose on the way. Each (page,
// head) has a power-of-two scale for its keys and one for its values: v = code *
// scale is exact in bf16, and a page whose scale grows by 2^n keeps its codes'
// mantissas.
#pragma once

#include "mga_common.hpp"

namespace mga {

constexpr int kScaleMin = -100, kScaleMax = 119;   // exponents: scaled codes are normal, finite bf16
constexpr int kMaxSeqs = 4096;

// Exponent of the least power of two of which 448 = 1.75 * 2^8 hold amax >= 0.
__device__ __forceinline__ int scale_exp(float amax) {
  const uint32_t u = __builtin_bit_cast(uint32_t, amax);
  const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffff) > 0x600000);
  return min(max(e, kScaleMin), kScaleMax);
}
__device__ __forceinline__ float pow2(int e) { return __builtin_bit_cast(float, (uint32_t)(e + 127) << 23); }
__device__ __forceinline__ int exp_of(float s) {
  return min(max((int)(__builtin_bit_cast(uint32_t, s) >> 23 & 255) - 127, kScaleMin), kScaleMax);
}

// The new tokens [first, first + n) of a sequence and its cached ones, whatever
// the caller's arrays hold within bounds.
struct SeqSpan {
  int first, n, len;
};
__device__ __forceinline__ SeqSpan seq_span(const int32_t *cu, const int32_t *lengths, int b, int T, int capacity) {
  SeqSpan s;
  s.first = min(max(cu[b], 0), T);
  s.n = min(max(cu[b + 1], s.first), T) - s.first;
  s.len = min(max(lengths[b], 0), capacity);
  return s;
}

}  // namespace mga
