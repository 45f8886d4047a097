// score.hpp -- what a score meets on its way to a weight.
#pragma once

#include <hip/hip_runtime.h>

namespace sts {

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// tanh to a few units in the last place relative to itself, also for small
// arguments: x P(x^2) below 0.6 (P fitted to tanh(x)/x at Chebyshev nodes, 9e-11),
// where 1 - 2/(e^2x + 1) would cancel; that form above.
__device__ __forceinline__ float tanh_rel(float x) {
  const float a = fabsf(x), z = x * x;
  float pz = 0.0022146995f;
  pz = fmaf(pz, z, -0.0082483031f);
  pz = fmaf(pz, z, 0.0217261855f);
  pz = fmaf(pz, z, -0.0539507493f);
  pz = fmaf(pz, z, 0.1333322972f);
  pz = fmaf(pz, z, -0.3333333135f);
  const float small = fmaf(x * z, pz, x);
  const float t = exp2_hw(a * (2.f * kLog2e));  // inf for large a: 2 / inf = 0
  const float big = copysignf(1.f - 2.f * __builtin_amdgcn_rcpf(t + 1.f), x);
  return a < 0.6f ? small : big;
}

}  // namespace sts
