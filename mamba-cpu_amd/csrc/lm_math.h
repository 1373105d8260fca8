// Scalar functions to about one unit in the last place of float32, for the
// kernels whose results are compared at that accuracy, and rows of any length
// in vectors of four elements.
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

// softplus(x), stable at both ends: log(1 + e) by v_log_f32 of u = 1 + e as
// rounded, times e / (u - 1), which takes the rounding back (Kahan's log1p); 20
// instructions where expf and log1pf take 100.
__device__ __forceinline__ float softplus_acc(float x) {
  const float e = exp_acc(-fabsf(x)), u = 1.0f + e;
  const float l = __builtin_amdgcn_logf(u) * kLn2 * (e * fast_rcp(u - 1.0f));
  return fmaxf(x, 0.f) + (u == 1.0f ? e : l);
}

// ---- four elements of a row, or what is left of it -----------------------------------

// n values (1 to 4) from element i on, as one vector where all four are there.
template <typename T> __device__ __forceinline__ void ld_upto4(const T* row, int64_t i, int n, float (&v)[4]) {
  if (n == 4) return ld4_elem<T>(row, i, v);
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = e < n ? to_f32(row[i + e]) : 0.f;
}
template <typename T> __device__ __forceinline__ void st_upto4(T* row, int64_t i, int n, const float (&v)[4]) {
  if (n == 4) return st4_elem<T>(row, i, v);
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (e < n) row[i + e] = from_f32<T>(v[e]);
}
__device__ __forceinline__ int upto4(int64_t left) { return left < 4 ? static_cast<int>(left) : 4; }

}  // namespace mcpu
