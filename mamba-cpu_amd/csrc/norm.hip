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
// A row of up to kNormMost elements is held in registers, four neighbouring
// elements a vector: by one wave (rows up to 1536), whose sums need no barrier,
// or by the four waves of a workgroup. The backward makes one pass: a workgroup
// takes every parts-th row, forms dz and adds to the parameters' gradients in
// its registers; the parts are then added in order. Longer rows are read again
// for each step by the norm_wide kernels, an element a load: 4096 x 12288 bf16 take
// 158 us forward and 152 + 71 backward, where their bytes take 39 and 59.
//
// Every sum is float32 in a fixed order. t is rounded before mean(t) is taken
// from it (no contraction), so that what cancels cancels exactly.
#include "launch.h"
#include "lm_params.h"
#include "lm_math.h"

namespace mcpu {
namespace {

constexpr int kThreads = 256;
constexpr int kGroupWaves = kThreads / 64;

__device__ __forceinline__ float wave_sum(float v) {
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
// Sum over the workgroup, in every thread; `slot` may be used again behind the
// next barrier.
__device__ __forceinline__ float group_sum(float v, float* slot) {
  v = wave_sum(v);
  if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = v;
  __syncthreads();
  return (slot[0] + slot[1]) + (slot[2] + slot[3]);
}

// ---- rows in registers: W waves a row, NV vectors a lane ----------------------------------

template <int W> __device__ __forceinline__ float row_sum(float v, float* slot) {
  return W == 1 ? wave_sum(v) : group_sum(v, slot);
}
// The first element of this lane's j-th vector.
template <int W> __device__ __forceinline__ int64_t column(int j) {
  return (j * 64 * W + (W == 1 ? threadIdx.x & 63 : threadIdx.x)) * 4ll;
}

template <typename T, typename R>
__device__ __forceinline__ void load_z4(const NormParams& p, int64_t row, int64_t i, int n, float (&z)[4]) {
  if (p.z != nullptr) return ld_upto4<float>(p.z + row * p.dim, i, n, z);
  ld_upto4<T>(static_cast<const T*>(p.x) + row * p.sx, i, n, z);
  if (p.residual != nullptr) {
    float r[4];
    ld_upto4<R>(static_cast<const R*>(p.residual) + row * p.sres, i, n, r);
#pragma unroll
    for (int e = 0; e < 4; ++e) z[e] += r[e];
  }
}

template <typename T, typename R, int W, int NV>
__global__ __launch_bounds__(kThreads) void norm_fwd_kernel(const NormParams p) {
  __shared__ float slots[3][kGroupWaves];
  const int64_t group = p.first + blockIdx.x;
  const int64_t row = W == 1 ? group * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : group;
  if (row >= p.rows) return;
  const float inv = 1.0f / static_cast<float>(p.dim);
  float z[NV][4] = {};
  int n[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int64_t i = column<W>(j);
    n[j] = i < p.dim ? upto4(p.dim - i) : 0;
    if (n[j] > 0) load_z4<T, R>(p, row, i, n[j], z[j]);
    if (n[j] > 0 && p.res_out != nullptr) st_upto4<R>(static_cast<R*>(p.res_out) + row * p.dim, i, n[j], z[j]);
  }
  float mean = 0.f;
  if (!p.rms) {
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) sum += (z[j][0] + z[j][1]) + (z[j][2] + z[j][3]);
    mean = row_sum<W>(sum, slots[0]) * inv;
  }
  // The mean's own rounding, up to 2^-24 of a mean far from zero, is the mean of
  // what is left (off).
  float sq = 0.f, rest = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      z[j][e] -= mean;
      const float c = e < n[j] ? z[j][e] : 0.f;
      sq = fmaf(c, c, sq);
      rest += c;
    }
  sq = row_sum<W>(sq, slots[1]) * inv;
  const float off = p.rms ? 0.f : row_sum<W>(rest, slots[2]) * inv;
  const float rstd = 1.0f / sqrtf(fmaf(-off, off, sq) + p.eps);
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    if (n[j] <= 0) continue;
    const int64_t i = column<W>(j);
    float w[4], b[4] = {}, y[4];
    ld_upto4<float>(p.weight, i, n[j], w);
    if (p.bias != nullptr) ld_upto4<float>(p.bias, i, n[j], b);
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = fmaf((z[j][e] - off) * rstd, w[e], b[e]);
    st_upto4<T>(static_cast<T*>(p.y) + row * p.sy, i, n[j], y);
  }
  if (W == 1 ? (threadIdx.x & 63) == 0 : threadIdx.x == 0) {
    if (p.mean != nullptr) p.mean[row] = mean + off;
    if (p.rstd != nullptr) p.rstd[row] = rstd;
  }
}

// BIAS: dbias too.
template <typename T, typename R, int W, int NV, bool BIAS>
__global__ __launch_bounds__(kThreads) void norm_bwd_kernel(const NormParams p) {
  constexpr int kRows = kGroupWaves / W;  // rows a workgroup takes at once
  __shared__ float slots[2][2][kGroupWaves];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const float inv = 1.0f / static_cast<float>(p.dim);
  float w[NV][4] = {}, dw[NV][4] = {}, db[BIAS ? NV : 1][4] = {};
  int n[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int64_t i = column<W>(j);
    n[j] = i < p.dim ? upto4(p.dim - i) : 0;
    if (n[j] > 0) ld_upto4<float>(p.weight, i, n[j], w[j]);
  }
  int buf = 0;
  for (int64_t row = blockIdx.x * int64_t{kRows} + (W == 1 ? wave : 0); row < p.rows; row += p.parts * kRows, buf ^= 1) {
    const float mean = p.rms ? 0.f : p.mean[row], rstd = p.rstd[row];
    float z[NV][4] = {}, g[NV][4] = {};
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (n[j] > 0) {
        ld_upto4<T>(static_cast<const T*>(p.dy) + row * p.sdy, column<W>(j), n[j], g[j]);
        load_z4<T, R>(p, row, column<W>(j), n[j], z[j]);
      }
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        z[j][e] = (z[j][e] - mean) * rstd;  // zhat; times g = 0 behind the row's end
        dw[j][e] = fmaf(g[j][e], z[j][e], dw[j][e]);
        if constexpr (BIAS) db[j][e] += g[j][e];
        g[j][e] = __fmul_rn(g[j][e], w[j][e]);
        s1 += g[j][e];
        s2 = fmaf(g[j][e], z[j][e], s2);
      }
    if constexpr (W == 1) {
      s1 = wave_sum(s1);
      s2 = wave_sum(s2);
    } else {
      s1 = wave_sum(s1);
      s2 = wave_sum(s2);
      if ((threadIdx.x & 63) == 0) {
        slots[buf][0][wave] = s1;
        slots[buf][1][wave] = s2;
      }
      __syncthreads();
      s1 = (slots[buf][0][0] + slots[buf][0][1]) + (slots[buf][0][2] + slots[buf][0][3]);
      s2 = (slots[buf][1][0] + slots[buf][1][1]) + (slots[buf][1][2] + slots[buf][1][3]);
    }
    const float m1 = p.rms ? 0.f : s1 * inv, m2 = s2 * inv;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (n[j] <= 0) continue;
      const int64_t i = column<W>(j);
      float dz[4], r[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) dz[e] = rstd * (g[j][e] - m1 - z[j][e] * m2);
      if (p.dres_out != nullptr) {
        ld_upto4<R>(static_cast<const R*>(p.dres_out) + row * p.dim, i, n[j], r);
#pragma unroll
        for (int e = 0; e < 4; ++e) dz[e] += r[e];
      }
      st_upto4<T>(static_cast<T*>(p.dx) + row * p.dim, i, n[j], dz);
      if (p.dres != nullptr) st_upto4<R>(static_cast<R*>(p.dres) + row * p.dim, i, n[j], dz);
    }
  }
  float* part = p.part + blockIdx.x * (BIAS ? 2ll : 1ll) * p.dim;
  if constexpr (W == 1) {
    // The four waves' sums, added in order.
    __shared__ float sums[kGroupWaves - 1][BIAS ? 2 : 1][NV * 256];
    if (wave > 0) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          sums[wave - 1][0][(j * 4 + e) * 64 + (threadIdx.x & 63)] = dw[j][e];
          if constexpr (BIAS) sums[wave - 1][1][(j * 4 + e) * 64 + (threadIdx.x & 63)] = db[j][e];
        }
    }
    __syncthreads();
    if (wave > 0) return;
    for (int v = 0; v < kGroupWaves - 1; ++v)
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          dw[j][e] += sums[v][0][(j * 4 + e) * 64 + threadIdx.x];
          if constexpr (BIAS) db[j][e] += sums[v][1][(j * 4 + e) * 64 + threadIdx.x];
        }
  }
#pragma unroll
  for (int j = 0; j < NV; ++j)
    if (n[j] > 0) {
      st_upto4<float>(part, column<W>(j), n[j], dw[j]);
      if constexpr (BIAS) st_upto4<float>(part + p.dim, column<W>(j), n[j], db[j]);
    }
}

constexpr int kReduceWaves = 16;

// dweight (blockIdx.y = 0) or dbias (1): every kReduceWaves-th part by one
// wave, then the waves' sums in order.
__global__ __launch_bounds__(64 * kReduceWaves) void norm_reduce_kernel(const NormParams p) {
  __shared__ float sums[kReduceWaves][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t i = blockIdx.x * 64ll + lane, kinds = gridDim.y;
  float sum = 0.f;
  if (i < p.dim) {
#pragma unroll 8
    for (int64_t k = wave; k < p.parts; k += kReduceWaves) sum += p.part[(k * kinds + blockIdx.y) * p.dim + i];
  }
  sums[wave][lane] = sum;
  __syncthreads();
  if (wave > 0 || i >= p.dim) return;
  for (int v = 1; v < kReduceWaves; ++v) sum += sums[v][lane];
  (blockIdx.y == 0 ? p.dweight : p.dbias)[i] = sum;
}

// ---- longer rows -----------------------------------------------------------------------------

template <typename T, typename R>
__device__ __forceinline__ float load_z(const NormParams& p, int64_t row, int64_t i) {
  if (p.z != nullptr) return p.z[row * p.dim + i];
  float z = ld<T>(p.x, row * p.sx + i);
  if (p.residual != nullptr) z += ld<R>(p.residual, row * p.sres + i);
  return z;
}

template <typename T, typename R> __global__ __launch_bounds__(kThreads) void norm_wide_fwd_kernel(const NormParams p) {
  __shared__ float slots[3][kThreads / 64];
  const int64_t row = p.first + blockIdx.x;
  float sum = 0.f;
  if (!p.rms)
    for (int64_t i = threadIdx.x; i < p.dim; i += kThreads) sum += load_z<T, R>(p, row, i);
  const float mean = p.rms ? 0.f : group_sum(sum, slots[0]) / p.dim;
  // As above: what the mean's rounding left is taken out of what is left (off).
  float sq = 0.f, rest = 0.f;
  for (int64_t i = threadIdx.x; i < p.dim; i += kThreads) {
    const float z = load_z<T, R>(p, row, i) - mean;
    sq = fmaf(z, z, sq);
    rest += z;
  }
  sq = group_sum(sq, slots[1]) / p.dim;
  const float off = p.rms ? 0.f : group_sum(rest, slots[2]) / p.dim;
  const float rstd = 1.0f / sqrtf(fmaf(-off, off, sq) + p.eps);
  for (int64_t i = threadIdx.x; i < p.dim; i += kThreads) {
    const float z = load_z<T, R>(p, row, i);
    const float y = (z - mean - off) * rstd * p.weight[i] + (p.bias == nullptr ? 0.f : p.bias[i]);
    st<T>(p.y, row * p.sy + i, y);
    if (p.res_out != nullptr) st<R>(p.res_out, row * p.dim + i, z);
  }
  if (threadIdx.x == 0) {
    if (p.mean != nullptr) p.mean[row] = mean + off;
    if (p.rstd != nullptr) p.rstd[row] = rstd;
  }
}

template <typename T, typename R> __global__ __launch_bounds__(kThreads) void norm_wide_dx_kernel(const NormParams p) {
  __shared__ float slots[2][kThreads / 64];
  const int64_t row = p.first + blockIdx.x;
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
template <typename T, typename R> __global__ __launch_bounds__(kThreads) void norm_wide_dw_kernel(const NormParams p) {
  const int64_t i = blockIdx.x * int64_t{kThreads} + threadIdx.x, part = blockIdx.y;
  if (i >= p.dim) return;
  float dw = 0.f, db = 0.f;
  for (int64_t row = part; row < p.rows; row += p.parts) {
    const float dy = ld<T>(p.dy, row * p.sdy + i);
    const float mean = p.rms ? 0.f : p.mean[row];
    dw = fmaf(dy, (load_z<T, R>(p, row, i) - mean) * p.rstd[row], dw);
    db += dy;
  }
  const int64_t kinds = p.dbias != nullptr ? 2 : 1;
  p.part[part * kinds * p.dim + i] = dw;
  if (kinds == 2) p.part[(part * kinds + 1) * p.dim + i] = db;
}

// f(x value, residual value) for the storage types of the call: the residual
// has x's type or float32.
template <typename F> void by_dtypes(const NormParams& p, F&& f) {
  const bool wide = p.res_dtype == MCPU_F32;
  if (p.x_dtype == MCPU_F32) f(float{}, float{});
  else if (p.x_dtype == MCPU_BF16) wide ? f(bf16{}, float{}) : f(bf16{}, bf16{});
  else wide ? f(f16{}, float{}) : f(f16{}, f16{});
}

// f(waves a row, vectors a lane) as constants, for rows of up to kNormMost.
template <typename F> void by_dim(int64_t dim, F&& f) {
  constexpr std::integral_constant<int, 1> one;
  constexpr std::integral_constant<int, 4> four;
  if (dim <= 256) f(one, std::integral_constant<int, 1>{});
  else if (dim <= 768) f(one, std::integral_constant<int, 3>{});
  else if (dim <= kNormWave) f(one, std::integral_constant<int, 6>{});
  else if (dim <= 3 * 1024) f(four, std::integral_constant<int, 3>{});
  else if (dim <= 5 * 1024) f(four, std::integral_constant<int, 5>{});
  else f(four, std::integral_constant<int, 8>{});
}

}  // namespace

int64_t norm_bwd_parts(int64_t rows, int64_t dim) {
  // As many workgroups as the registers of a row length let a CU hold at once:
  // more would take turns, and each costs 4 or 8 bytes a column to write and read.
  // 1763 x 8034 bf16 with float32 residual: 67 us with two a CU, 90 with four;
  // 4096 x 4096: 63 with three, 81 with four, 75 with two; 16384 x 2560: 135 with
  // four, 151 with three.
  const int64_t per_cu = dim <= 3 * 1024 ? 4 : dim <= 5 * 1024 ? 3 : 2;
  const int64_t most = dim > kNormMost ? 64 : 256 * per_cu, at_once = dim <= kNormWave ? 4 : 1;
  const int64_t groups = (rows + at_once - 1) / at_once;
  return groups < 1 ? 1 : groups < most ? groups : most;
}

hipError_t norm_fwd_launch(NormParams p, hipStream_t st) {
  by_dtypes(p, [&](auto t, auto r) {
    using T = decltype(t);
    using R = decltype(r);
    if (p.dim > kNormMost) {
      launch_all(p.rows, kThreads, [&](int64_t first, unsigned groups) {
        p.first = first;
        hipLaunchKernelGGL((norm_wide_fwd_kernel<T, R>), dim3(groups), dim3(kThreads), 0, st, p);
      });
      return;
    }
    by_dim(p.dim, [&](auto w, auto nv) {
      constexpr int W = decltype(w)::value, NV = decltype(nv)::value;
      launch_all((p.rows * W + 3) / 4, kThreads, [&](int64_t first, unsigned groups) {
        p.first = first;
        hipLaunchKernelGGL((norm_fwd_kernel<T, R, W, NV>), dim3(groups), dim3(kThreads), 0, st, p);
      });
    });
  });
  return hipGetLastError();
}

hipError_t norm_bwd_launch(NormParams p, hipStream_t st) {
  const unsigned kinds = p.dbias != nullptr ? 2 : 1;
  by_dtypes(p, [&](auto t, auto r) {
    using T = decltype(t);
    using R = decltype(r);
    if (p.dim > kNormMost) {
      launch_all(p.rows, kThreads, [&](int64_t first, unsigned groups) {
        p.first = first;
        hipLaunchKernelGGL((norm_wide_dx_kernel<T, R>), dim3(groups), dim3(kThreads), 0, st, p);
      });
      hipLaunchKernelGGL((norm_wide_dw_kernel<T, R>),
                         dim3(static_cast<unsigned>((p.dim + kThreads - 1) / kThreads), static_cast<unsigned>(p.parts)),
                         dim3(kThreads), 0, st, p);
      return;
    }
    by_dim(p.dim, [&](auto w, auto nv) {
      constexpr int W = decltype(w)::value, NV = decltype(nv)::value;
      const dim3 grid(static_cast<unsigned>(p.parts)), block(kThreads);
      if (kinds == 2) hipLaunchKernelGGL((norm_bwd_kernel<T, R, W, NV, true>), grid, block, 0, st, p);
      else hipLaunchKernelGGL((norm_bwd_kernel<T, R, W, NV, false>), grid, block, 0, st, p);
    });
  });
  hipLaunchKernelGGL(norm_reduce_kernel, dim3(static_cast<unsigned>((p.dim + 63) / 64), kinds),
                     dim3(64 * kReduceWaves), 0, st, p);
  return hipGetLastError();
}

}  // namespace mcpu
