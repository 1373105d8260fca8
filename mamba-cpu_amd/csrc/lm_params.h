// Kernel parameter blocks of the residual norm, the embedding and the token
// sampler, shared by the kernels and the C-ABI layer that fills them.
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

namespace mcpu {

struct NormParams {
  const void* x;         // (rows, dim), row stride sx
  const void* residual;  // (rows, dim), row stride sres, or null
  const float* z;     // backward: x + residual, contiguous, instead of the two; or null
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
  float* part;   // (parts, 1 or, with dbias, 2, dim): dweight and dbias partials
  int64_t rows, dim, parts;
  int64_t first;  // this launch's first workgroup
  int64_t sx, sres, sy, sdy;
  float eps;
  int rms;
  int x_dtype, res_dtype;
};

constexpr int64_t kNormWave = 1536;  // longest row of one wave
constexpr int64_t kNormMost = 8192;  // longest row held in registers
// Workgroups of the backward: each leaves one partial of dweight and dbias.
int64_t norm_bwd_parts(int64_t rows, int64_t dim);
hipError_t norm_fwd_launch(NormParams p, hipStream_t st);
hipError_t norm_bwd_launch(NormParams p, hipStream_t st);

struct EmbeddingParams {
  const void* ids;  // (tokens) int32 or int64
  int ids64;
  const void* weight;  // (vocab, dim), row stride sw
  void* out;           // (tokens, dim) contiguous
  const void* dout;    // (tokens, dim), row stride sdo
  void* dweight;       // (vocab, dim) contiguous
  int32_t* order;      // token positions sorted by id, in token order within an id
  int32_t* start;      // (vocab + 1): where each id's positions start in `order`
  float* part;         // (chunks, 2, dim): partial sums of ids that cross a chunk's edge
  int64_t tokens, vocab, dim, sw, sdo;
  int64_t first;  // this launch's first workgroup
  float scale;
  int dtype;
};

constexpr int kEmbedChunk = 32;  // sorted positions per workgroup (at most 64: one per lane)
int64_t embedding_chunks(int64_t tokens);
hipError_t embedding_fwd_launch(EmbeddingParams p, hipStream_t st);
hipError_t embedding_bwd_launch(EmbeddingParams p, hipStream_t st);

struct SampleParams {
  const void* logits;  // (rows, vocab), row stride sl
  const float* noise;  // (rows, vocab), row stride sn, or null
  // One setting for all rows, or one per row where the pointer is given.
  float temperature, top_p, min_p;
  int32_t top_k;
  const float* temperature_rows;
  const float* top_p_rows;
  const float* min_p_rows;
  const int32_t* top_k_rows;
  int64_t* token;   // (rows)
  float* logprob;   // (rows), or null
  void* slices;  // what the slices of uncut rows leave (sample_workspace bytes)
  int64_t rows, vocab, sl, sn;
  int64_t first;  // this launch's first workgroup
  int dtype;
};

constexpr int kSampleSlice = 8192;  // logits of a slice
int64_t sample_slices(const SampleParams& p);
size_t sample_workspace(const SampleParams& p);
hipError_t sample_launch(SampleParams p, hipStream_t st);

}  // namespace mcpu
