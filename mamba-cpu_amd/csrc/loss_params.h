// Kernel parameter block of the head's losses, shared by the kernels and the
// C-ABI layer that fills it.
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

#include "mamba_hip.h"

namespace mcpu {

// What one call passes between its kernels on the GPU.
struct LossScalars {
  int32_t kept;          // rows that count
  uint32_t hmax, wmax;   // the largest finite magnitudes, as bits: float32 operands; hidden in f16 for dweight
  int32_t hsplit;        // backward: splits of dhidden's products
  float unit;            // backward: the largest unit of a row's ds
};

struct LossParams {
  const void* hidden;    // (tokens, dim), row stride sh
  const void* weight;    // (vocab, dim), row stride sw
  const void* ids;       // (tokens, k) int32 or int64
  const float* teacher;  // (tokens, k), or null: cross entropy
  int ids64;
  int64_t tokens, vocab, dim, k, sh, sw, ignore;
  float temperature;
  int dtype, reduction;
  float* loss;    // (tokens), or (1) where reduced
  float* each;    // (tokens): loss, or the terms of the reduced one
  float* lse;     // (tokens)
  float* picked;  // distillation: (tokens, k), the products of hidden with the ids' rows; else workspace, (padded
                  // tokens), the targets' in the order of `rows` (few tokens: as they come)
  float* stat;    // (4, tokens) in the order of `rows`: maximum, sum of exp(c (s - it)), a target's share of it,
                  // the others'
  float* share;   // (tokens, k): the teacher's distribution, or null
  int32_t* rows;  // (tokens + 1): the rows that count in order, then the others; then how many count
  uint32_t* laid;      // float32: wmax beside wrows, where both are kept for the backward; or null
  // backward
  const float* dloss;  // (tokens), or (1) where reduced
  const float* dlse;   // (tokens), or null
  void* dhidden;       // (tokens, dim) contiguous, or null
  void* dweight;       // (vocab, dim) contiguous, or null
  // workspace
  LossScalars* scal;
  uint8_t* keep;      // (tokens)
  int32_t* target;    // (padded tokens) in the order of `rows`, cross entropy; else null
  float* cross;       // (tokens): sum of q (log q - c s)
  float2* part;       // (vocab parts, padded tokens; few tokens: whole 16, 32 or 64): maximum of each part and
                      // sum of exp(c (s - it))
  float* coef;        // (4, padded tokens): factor of 2^(logit - maximum), the target's ds or the shares' factor,
                      // the maximum, the unit of ds (0: the largest)
  void* hrows;        // (pieces, padded tokens, padded dim): hidden's rows that count
  void* hscaled;      // hidden's rows in the largest unit, or null: one unit for all (distillation, but for rows'
                      // gradients in f16 pieces)
  void* wrows;        // (pieces, vocab, padded dim), which may be of `laid`, or null: weight is read in place
  void* grad;         // (pieces, padded tokens, vocab piece): gradients of the logits
  float* acc;         // (splits, rows that count, padded, padded dim): gradient of hidden
  float* dwpart;      // (splits, vocab piece, padded dim), or null: gradient of weight in one go
  int64_t tpad, dpad, vpiece;
  int64_t vrows;      // of this piece, a multiple of 256, at most vpiece
  int64_t htiles;     // most tiles of 256 x 256 of dhidden's products, splits counted
  int wsplit;
  int blocks;         // logits by blocks of 64 tokens and 128 vocabulary rows
  int few_lds;        // hidden's and weight's rows are 16-byte aligned
  int64_t first;      // this launch's first workgroup
};

constexpr int kLossTile = 256;   // rows and columns of a workgroup's tile of a product
constexpr int kLossDepth = 64;   // terms of a tile that are in LDS at once
constexpr int kLossPart = 128;   // vocabulary rows of one maximum and sum, and of a block
constexpr int kLossFew = 64;     // tokens of a block; up to so many in all, the weight streams past them
constexpr int kLossBlocks = 512;  // most blocks taken instead of tiles
constexpr int kLossMostSplits = 64;
constexpr int64_t kLossSplitTiles = 1536;  // most results of a split product, of 256 KiB each
constexpr int64_t kLossMaxK = 1024;

// float32 operands are two f16 pieces.
inline int loss_pieces(int dtype) { return dtype == MCPU_F32 ? 2 : 1; }
// Sets the padded sizes, the vocabulary piece and the splits (wsplit: the most of any piece); what a piece
// that begins at vp has of them.
void loss_plan(LossParams& p);
int64_t loss_piece_rows(const LossParams& p, int64_t vp);
int loss_wsplit(const LossParams& p, int64_t vp);
hipError_t loss_zero(void* at, int64_t bytes, hipStream_t st);
hipError_t loss_fwd_launch(LossParams p, hipStream_t st);
hipError_t loss_bwd_launch(LossParams p, hipStream_t st);

}  // namespace mcpu
