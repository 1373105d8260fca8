// Scalar functions to about one unit in the last place of float32, for the
// kernels whose results are compared at that accuracy.
#pragma once

#include "mcpu_common.h"

namespace mcpu {

// exp(x) over the whole range: the rounding error of x * log2(e) is carried
// along (v_exp_f32 alone loses |x| ulp). Clamped where the result leaves the
// normal range, so that infinities stay exact; NaN passes through.
__device__ __forceinline__ float exp_acc(float x) {
  x = x > 88.f ? 88.f : (x < -104.f ? -104.f : x);
  const float t = x * kLog2e;
  const float lo = fmaf(x, kLog2e, -t) + x * 1.925963033500e-8f;  // log2(e) - float(log2(e))
  const float e = fast_exp2(t);
  return fmaf(e, lo * kLn2, e);
}

// sigmoid(x) and 1 - sigmoid(x) from one exponential, each to its own ulp.
__device__ __forceinline__ float sigmoid_acc(float x, float& one_minus) {
  const float e = exp_acc(-x);
  const float s = fast_rcp(1.0f + e);
  one_minus = e * s;
  return s;
}

// softplus(x), stable at both ends.
__device__ __forceinline__ float softplus_acc(float x) { return fmaxf(x, 0.f) + log1pf(expf(-fabsf(x))); }

}  // namespace mcpu
