// Kernel parameter blocks of the residual norm, the embedding and the token
// sampler, shared by the kernels and the C-ABI layer that fills them.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace mcpu {

struct NormParams {
  const void* x;         // (rows, dim), row stride sx
  const void* residual;  // (rows, dim), row stride sres, or null
  const float* weight;
  const float* bias;  // or null
  void* y;            // (rows, dim), row stride sy
  void* res_out;      // (rows, dim) contiguous, or null
  float* mean;        // (rows), layer norm only
  float* rstd;        // (rows)
  const void* dy;
  const void* dres_out;  // contiguous, or null
  void* dx;              // contiguous
  void* dres;            // contiguous, or null
  float* dweight;
  float* dbias;  // or null
  float* part;   // (parts, 1 or 2, dim): dweight and dbias partials
  int64_t rows, dim, parts;
  int64_t sx, sres, sy, sdy;
  float eps;
  int rms;
  int x_dtype, res_dtype;
};

// Workgroups of the backward: each leaves one partial of dweight and dbias.
int64_t norm_bwd_parts(int64_t rows, int64_t dim);
hipError_t norm_fwd_launch(const NormParams& p, hipStream_t st);
hipError_t norm_bwd_launch(const NormParams& p, hipStream_t st);

}  // namespace mcpu
