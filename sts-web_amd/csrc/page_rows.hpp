// page_rows.hpp -- device code shared by the kernels over paged K/V rows.
#pragma once

#include <cfloat>

#include "pages.hpp"
#include "sts_attn.h"

namespace sts {

// Rows of stream b.
__device__ __forceinline__ uint32_t paged_len(const PagedRows& p, uint32_t b) {
  const int32_t n = p.lens[b];
  return n <= 0 ? 0u : min((uint32_t)n, p.max_rows);
}

// Row r of stream b, head j as a row index into k, v and their scales; false where no
// page holds it.
__device__ __forceinline__ bool paged_row(const PagedRows& p, uint32_t b, uint32_t j, uint32_t r, uint64_t& at) {
  const uint32_t page = (uint32_t)p.table[(uint64_t)b * p.max_pages + (r >> p.shift)];
  at = (((uint64_t)page * p.KH + j) << p.shift) + (r & ((1u << p.shift) - 1));
  return page < p.pages;
}

// 8-bit rows.  A row is kept as codes c in -127..127 and one f32 scale s, the value
// being c s: s = max|x| / 127 rounded to f32, c the whole number nearest to x / s (of
// two, the even one).
//
// The row's scale; rows whose largest value is below 2^-64 are kept as zeros (their scale
// times an attention weight would lose bits to f32's lower end), rows with an infinity or
// NaN as NaN.
__device__ __forceinline__ float row_scale(float top) {
  if (!(top <= FLT_MAX)) return __builtin_nanf("");
  return top < 0x1p-64f ? 0.f : top / 127.f;
}

// The code of x under scale s (by = 1 / s, rounded): x by, rounded, is at most one
// step off; what it leaves of x is exact in f32 (x itself below s / 2, else a
// difference of multiples of a unit of s, or of x between s / 2 and s) and says whether
// the next code is nearer.
__device__ __forceinline__ int row_code(float x, float s, float by) {
  const float c = rintf(x * by);
  const float left = fmaf(-c, s, x), half = 0.5f * s;
  int code = (int)c;
  if (left > half || (left == half && (code & 1))) ++code;
  else if (left < -half || (left == -half && (code & 1))) --code;
  return min(max(code, -127), 127);
}

// Four codes, the first in the low byte; zeros for a row without a scale.
__device__ __forceinline__ uint32_t row_codes(float4 x, float s) {
  if (!(s > 0.f)) return 0u;
  const float by = 1.f / s;
  return ((uint32_t)row_code(x.x, s, by) & 255u) | ((uint32_t)row_code(x.y, s, by) & 255u) << 8 |
         ((uint32_t)row_code(x.z, s, by) & 255u) << 16 | (uint32_t)row_code(x.w, s, by) << 24;
}

__device__ __forceinline__ uint2 bf16x4(float4 x) {
  typedef __bf16 b4 __attribute__((ext_vector_type(4)));
  const b4 y = {(__bf16)x.x, (__bf16)x.y, (__bf16)x.z, (__bf16)x.w};
  return __builtin_bit_cast(uint2, y);
}

// The largest magnitude; a NaN stays (fmaxf would drop it).
__device__ __forceinline__ float largest(float4 x) {
  return __builtin_elementwise_maximum(__builtin_elementwise_maximum(fabsf(x.x), fabsf(x.y)),
                                       __builtin_elementwise_maximum(fabsf(x.z), fabsf(x.w)));
}

// The largest magnitude of the G lanes' values (G consecutive lanes, a power of two).
template <int G>
__device__ __forceinline__ float lanes_largest(float4 x) {
  float top = largest(x);
#pragma unroll
  for (int d = 1; d < G; d *= 2) top = __builtin_elementwise_maximum(top, __shfl_xor(top, d, G));
  return top;
}

}  // namespace sts
