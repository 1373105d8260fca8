// Kernel parameter blocks and launch shapes of the gated linear recurrence,
// shared by the kernels and the C-ABI layer that fills them.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace mcpu {

constexpr int kGatedT = 16;  // steps of a wave's segment: the forward keeps the state before each
// Waves of a workgroup, with one segment of its chunk each. The backward
// holds twice the registers: with 4 waves four of its workgroups share a CU
// instead of two (87 against 98 us for 8 x 2048 x 1536 bf16, 158 against 161 for
// 16384 x 2560). The forward has three or more either way, and longer chunks
// look back less (105 against 114 us for 16384 x 2560).
constexpr int kGatedFwdWaves = 8, kGatedBwdWaves = 4;

struct GatedScanParams {
  const void* x;
  const void* a_gate;
  const void* x_gate;
  const float* decay;
  const float* init;
  const int32_t* seq_idx;  // (batch, len) contiguous, or null
  void* y;
  float* last;
  float* ckpt;  // (batch, ceil(len / kGatedT), dim)
  const void* dy;
  const float* dlast;
  void* dx;
  void* da_gate;
  void* dx_gate;
  float* ddecay;
  float* ddecay_part;  // (batch, chunks, dim) partial sums over time
  // Zeroed before the launch, with more than one chunk: the tickets handed out
  // for each tile of each row, and (batch, chunks, dim) what a chunk has published.
  uint32_t* tickets;
  uint64_t* records;
  float* dinit;
  int64_t batch, len, dim;
  int64_t chunks;
  int64_t first;  // this launch's first workgroup
  float c;
  int64_t sx[3], sa[3], si[3], sy[3], sdy[3], sdx[3], sda[3], sdi[3];  // (batch, len, dim)
};

struct GatedStepParams {
  float* state;
  const void* x;
  const void* a_gate;
  const void* x_gate;
  const float* decay;
  void* y;
  int64_t batch, dim;
  int64_t first;  // this launch's first workgroup
  float c;
  int64_t sst[2], sx[2], sa[2], si[2];
  const int32_t* state_idx;  // state row per batch row, or null
  int64_t state_batch;
};

hipError_t gated_scan_fwd_launch(GatedScanParams p, int dtype, hipStream_t st);
hipError_t gated_scan_bwd_launch(GatedScanParams p, int dtype, hipStream_t st);
hipError_t gated_edge_launch(const float* from, float* to, int64_t n, hipStream_t st);
hipError_t gated_step_launch(GatedStepParams p, int dtype, hipStream_t st);

}  // namespace mcpu
