// page_rows.hpp -- device code shared by the kernels over paged K/V rows.
#pragma once

#include <cfloat>

#include "lane.hpp"
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
// NaN as NaN.  The quotient is the product with 1 / 127, half an ulp and a sixteenth off at
// most, and one correction by what it leaves, which rounds it right (Markstein 1990).
__device__ __forceinline__ float row_scale(float top) {
  constexpr float by = 1.f / 127.f;
  const float s = top * by, right = fmaf(fmaf(-s, 127.f, top), by, s);
  if (!(top <= FLT_MAX)) return __builtin_nanf("");
  return top < 0x1p-64f ? 0.f : right;
}

// The code of x under scale s: c is at most one step off; what it leaves of x is exact in
// f32 (x itself below s / 2, else a difference of multiples of a unit of s, or of x between
// s / 2 and s) and says whether the next code is nearer.
__device__ __forceinline__ int nearer_code(float x, float s, int c) {
  const float left = fmaf(-(float)c, s, x), half = 0.5f * s;
  if (left > half || (left == half && (c & 1))) ++c;
  else if (left < -half || (left == -half && (c & 1))) --c;
  return min(max(c, -127), 127);
}

// Four codes, the first in the low byte; zeros for a row without a scale.  Adding 1.5 2^23
// leaves the whole number in the float's low bits; where it leaves less than half a step of
// x, as nearly always, it is the code.
__device__ __forceinline__ uint32_t row_codes(float4 x, float s) {
  if (!(s > 0.f)) return 0u;
  const float by = __builtin_amdgcn_rcpf(s), half = 0.5f * s;
  const float in[4] = {x.x, x.y, x.z, x.w};
  uint32_t c[4];
  bool sure = true;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float y = fmaf(in[i], by, 0x1.8p23f);
    sure &= fabsf(fmaf(0x1.8p23f - y, s, in[i])) < half;
    c[i] = __float_as_uint(y);
  }
  if (!sure) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      c[i] = (uint32_t)nearer_code(in[i], s, (int)(__uint_as_float(c[i]) - 0x1.8p23f));
  }
  return __builtin_amdgcn_perm(__builtin_amdgcn_perm(c[3], c[2], 0x0c0c0400),
                               __builtin_amdgcn_perm(c[1], c[0], 0x0c0c0400), 0x05040100);
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

// The largest of the G lanes' magnitudes (G consecutive lanes, a power of two up to 32).
template <int G, int LEVEL = 0>
__device__ __forceinline__ float lanes_largest(float top) {
  if constexpr ((1 << LEVEL) < G)
    return lanes_largest<G, LEVEL + 1>(__builtin_elementwise_maximum(top, xchg<LEVEL>(top)));
  return top;
}

}  // namespace sts
