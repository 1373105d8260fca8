// Residual norm on gfx950: forward and backward of
//
//   z = x + residual                      (float32, residual optional)
//   layer norm:  y = (z - mean) rstd w + b      rstd = 1 / sqrt(var + eps)
//   RMS norm:    y = z rstd w + b               rstd = 1 / sqrt(mean(z^2) + eps)
//
// with mean and var over a row, the variance from the centred values (two
// passes over registers or cache, not E[z^2] - E[z]^2). res_out is z rounded
// to the residual's type; y comes from the unrounded sum. Backward, with
// zhat = (z - mean) rstd (or z rstd) and t = w dy:
//
//   dz = rstd (t - mean(t) - zhat mean(t zhat)) + dres_out     (no mean(t) for RMS)
//   dweight = sum_rows dy zhat      dbias = sum_rows dy
//
// Every sum is float32 in a fixed order. t is rounded before mean(t) is taken
// from it (no contraction), so that what cancels cancels exactly.
#include "lm_params.h"
#include "mcpu_common.h"

namespace mcpu {
namespace {

constexpr int kThreads = 256;

// Sum over the workgroup, in every thread. `slot` (kThreads / 64 floats) may
// be reused after the next barrier.
__device__ __forceinline__ float group_sum(float v, float* slot) {
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = 0.f;
  for (int i = 0; i < kThreads / 64; ++i) s += slot[i];
  return s;
}

template <typename T, typename R>
__device__ __forceinline__ float load_z(const NormParams& p, int64_t row, int64_t i) {
  float z = ld<T>(p.x, row * p.sx + i);
  if (p.residual != nullptr) z += ld<R>(p.residual, row * p.sres + i);
  return z;
}

template <typename T, typename R> __global__ __launch_bounds__(kThreads) void norm_fwd_kernel(const NormParams p) {
  __shared__ float slots[2][kThreads / 64];
  const int64_t row = blockIdx.x;
  float sum = 0.f;
  if (!p.rms)
    for (int64_t i = threadIdx.x; i < p.dim; i += kThreads) sum += load_z<T, R>(p, row, i);
  const float mean = p.rms ? 0.f : group_sum(sum, slots[0]) / p.dim;
  float sq = 0.f;
  for (int64_t i = threadIdx.x; i < p.dim; i += kThreads) {
    const float z = load_z<T, R>(p, row, i) - mean;
    sq = fmaf(z, z, sq);
  }
  const float rstd = 1.0f / sqrtf(group_sum(sq, slots[1]) / p.dim + p.eps);
  for (int64_t i = threadIdx.x; i < p.dim; i += kThreads) {
    const float z = load_z<T, R>(p, row, i);
    const float y = (z - mean) * rstd * p.weight[i] + (p.bias == nullptr ? 0.f : p.bias[i]);
    st<T>(p.y, row * p.sy + i, y);
    if (p.res_out != nullptr) st<R>(p.res_out, row * p.dim + i, z);
  }
  if (threadIdx.x == 0) {
    if (p.mean != nullptr) p.mean[row] = mean;
    if (p.rstd != nullptr) p.rstd[row] = rstd;
  }
}

template <typename T, typename R> __global__ __launch_bounds__(kThreads) void norm_dx_kernel(const NormParams p) {
  __shared__ float slots[2][kThreads / 64];
  const int64_t row = blockIdx.x;
  const float mean = p.rms ? 0.f : p.mean[row], rstd = p.rstd[row];
  float s1 = 0.f, s2 = 0.f;
  for (int64_t i = threadIdx.x; i < p.dim; i += kThreads) {
    const float t = __fmul_rn(p.weight[i], ld<T>(p.dy, row * p.sdy + i));
    s1 += t;
    s2 = fmaf(t, (load_z<T, R>(p, row, i) - mean) * rstd, s2);
  }
  const float m1 = p.rms ? 0.f : group_sum(s1, slots[0]) / p.dim;
  const float m2 = group_sum(s2, slots[1]) / p.dim;
  for (int64_t i = threadIdx.x; i < p.dim; i += kThreads) {
    const float zh = (load_z<T, R>(p, row, i) - mean) * rstd;
    float dz = rstd * (__fmul_rn(p.weight[i], ld<T>(p.dy, row * p.sdy + i)) - m1 - zh * m2);
    if (p.dres_out != nullptr) dz += ld<R>(p.dres_out, row * p.dim + i);
    st<T>(p.dx, row * p.dim + i, dz);
    if (p.dres != nullptr) st<R>(p.dres, row * p.dim + i, dz);
  }
}

// Partial sums of dweight and dbias over the rows part, part + parts, ...
template <typename T, typename R> __global__ __launch_bounds__(kThreads) void norm_dw_kernel(const NormParams p) {
  const int64_t i = blockIdx.x * int64_t{kThreads} + threadIdx.x, part = blockIdx.y;
  if (i >= p.dim) return;
  float dw = 0.f, db = 0.f;
  for (int64_t row = part; row < p.rows; row += p.parts) {
    const float dy = ld<T>(p.dy, row * p.sdy + i);
    const float mean = p.rms ? 0.f : p.mean[row];
    dw = fmaf(dy, (load_z<T, R>(p, row, i) - mean) * p.rstd[row], dw);
    db += dy;
  }
  p.part[(part * 2) * p.dim + i] = dw;
  p.part[(part * 2 + 1) * p.dim + i] = db;
}

__global__ __launch_bounds__(kThreads) void norm_reduce_kernel(const NormParams p) {
  const int64_t i = blockIdx.x * int64_t{kThreads} + threadIdx.x;
  if (i >= p.dim) return;
  float dw = 0.f, db = 0.f;
  for (int64_t k = 0; k < p.parts; ++k) {
    dw += p.part[(k * 2) * p.dim + i];
    db += p.part[(k * 2 + 1) * p.dim + i];
  }
  p.dweight[i] = dw;
  if (p.dbias != nullptr) p.dbias[i] = db;
}

// f(x value, residual value) for the storage types of the call: the residual
// has x's type or float32.
template <typename F> void by_dtypes(const NormParams& p, F&& f) {
  const bool wide = p.res_dtype == MCPU_F32;
  if (p.x_dtype == MCPU_F32) f(float{}, float{});
  else if (p.x_dtype == MCPU_BF16) wide ? f(bf16{}, float{}) : f(bf16{}, bf16{});
  else wide ? f(f16{}, float{}) : f(f16{}, f16{});
}

}  // namespace

int64_t norm_bwd_parts(int64_t rows, int64_t) { return rows < 64 ? (rows < 1 ? 1 : rows) : 64; }

hipError_t norm_fwd_launch(const NormParams& p, hipStream_t st) {
  by_dtypes(p, [&](auto t, auto r) {
    hipLaunchKernelGGL((norm_fwd_kernel<decltype(t), decltype(r)>), dim3(static_cast<unsigned>(p.rows)),
                       dim3(kThreads), 0, st, p);
  });
  return hipGetLastError();
}

hipError_t norm_bwd_launch(const NormParams& p, hipStream_t st) {
  const unsigned cols = static_cast<unsigned>((p.dim + kThreads - 1) / kThreads);
  by_dtypes(p, [&](auto t, auto r) {
    using T = decltype(t);
    using R = decltype(r);
    if (p.rows > 0)
      hipLaunchKernelGGL((norm_dx_kernel<T, R>), dim3(static_cast<unsigned>(p.rows)), dim3(kThreads), 0, st,
                         p);
    hipLaunchKernelGGL((norm_dw_kernel<T, R>), dim3(cols, static_cast<unsigned>(p.parts)), dim3(kThreads), 0, st, p);
  });
  hipLaunchKernelGGL(norm_reduce_kernel, dim3(cols), dim3(kThreads), 0, st, p);
  return hipGetLastError();
}

}  // namespace mcpu
