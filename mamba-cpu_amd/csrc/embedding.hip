// Embedding on gfx950: out_t = scale weight[id_t], and its gradient
// dweight_v = scale sum_{t: id_t = v} dout_t.
//
// The gradient is a segmented sum over the tokens sorted by id: the sum of an
// id runs over its tokens in their order, in float32, and is rounded once, so
// the result does not depend on timing (no floating atomics). The sort needs
// one launch: a workgroup owns a range of ids, reads every token's id and so
// knows both how many tokens lie below its range (where its part of the order
// starts) and its own tokens; nothing passes between workgroups. An id outside
// the vocabulary has a zero row and no gradient.
#include "lm_params.h"
#include "mcpu_common.h"

namespace mcpu {
namespace {

__device__ __forceinline__ int64_t id_at(const EmbeddingParams& p, int64_t t) {
  return p.ids64 ? static_cast<const int64_t*>(p.ids)[t] : static_cast<const int32_t*>(p.ids)[t];
}

template <typename T> __global__ __launch_bounds__(256) void embedding_fwd_kernel(const EmbeddingParams p) {
  const int64_t t = blockIdx.x;
  const int64_t id = id_at(p, t);
  const bool in = id >= 0 && id < p.vocab;
  for (int64_t i = threadIdx.x; i < p.dim; i += 256)
    st<T>(p.out, t * p.dim + i, in ? ld<T>(p.weight, id * p.sw + i) * p.scale : 0.f);
}

constexpr int kSortWaves = 16;
constexpr int kSortIds = 512;  // most ids of one workgroup's range

__global__ __launch_bounds__(64 * kSortWaves) void embedding_sort_kernel(const EmbeddingParams p, int range) {
  __shared__ int count[kSortWaves][kSortIds];  // tokens of (wave, id), then where the next one goes
  __shared__ int below[kSortWaves], sums[kSortWaves];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t lo = blockIdx.x * int64_t{range};
  const int64_t hi = lo + range < p.vocab ? lo + range : p.vocab;
  const int n = static_cast<int>(hi - lo);
  for (int i = threadIdx.x; i < kSortWaves * kSortIds; i += 64 * kSortWaves) (&count[0][0])[i] = 0;
  __syncthreads();
  // A wave takes a run of the tokens, 64 at a time. Lanes with the same id of
  // the range find each other by ballot, one id after the other.
  const int64_t run = ((p.tokens + kSortWaves - 1) / kSortWaves + 63) / 64 * 64;
  const int64_t t0 = w * run, t1 = t0 + run < p.tokens ? t0 + run : p.tokens;
  int under = 0;
  for (int pass = 0; pass < 2; ++pass) {
    for (int64_t t = t0 + lane; t - lane < t1; t += 64) {
      const int64_t id = t < t1 ? id_at(p, t) : -1;
      const bool in = id >= lo && id < hi;
      const int slot = in ? static_cast<int>(id - lo) : -1;
      if (pass == 0) under += __popcll(__ballot(id >= 0 && id < lo));
      uint64_t left = __ballot(in);
      while (left != 0) {
        const int lead = __builtin_ctzll(left);
        const int s = __builtin_amdgcn_readlane(slot, lead);
        const uint64_t same = __ballot(slot == s);
        int first = 0;
        if (lane == lead) first = atomicAdd(&count[w][s], __popcll(same));
        if (pass == 1) {
          first = __builtin_amdgcn_readlane(first, lead);
          if (slot == s) p.order[first + __popcll(same & ((1ull << lane) - 1))] = static_cast<int32_t>(t);
        }
        left &= ~same;
      }
    }
    if (pass == 1) break;
    if (lane == 0) below[w] = under;
    __syncthreads();
    // Where each id starts: the tokens below the range, those of smaller ids
    // of the range (a scan over the workgroup), those of earlier waves.
    int total = 0;
    if (static_cast<int>(threadIdx.x) < n)
      for (int v = 0; v < kSortWaves; ++v) total += count[v][threadIdx.x];
    int incl = total;
    for (int o = 1; o < 64; o <<= 1) {
      const int up = __shfl_up(incl, o);
      if (lane >= o) incl += up;
    }
    if (lane == 63) sums[w] = incl;
    __syncthreads();
    int at = incl - total;
    for (int v = 0; v < kSortWaves; ++v) {
      at += below[v];
      if (v < w) at += sums[v];
    }
    if (static_cast<int>(threadIdx.x) < n) {
      p.start[lo + threadIdx.x] = at;
      if (lo + threadIdx.x == p.vocab - 1) p.start[p.vocab] = at + total;
      for (int v = 0; v < kSortWaves; ++v) {
        const int c = count[v][threadIdx.x];
        count[v][threadIdx.x] = at;
        at += c;
      }
    }
    __syncthreads();
  }
}

// One wave per row of dweight.
template <typename T> __global__ __launch_bounds__(256) void embedding_dw_kernel(const EmbeddingParams p) {
  const int lane = threadIdx.x & 63;
  const int64_t v = blockIdx.x * 4ll + (threadIdx.x >> 6);
  if (v >= p.vocab) return;
  const int s0 = p.start[v], s1 = p.start[v + 1];
  for (int64_t i = lane; i < p.dim; i += 64) {
    float sum = 0.f;
    for (int s = s0; s < s1; ++s) sum += ld<T>(p.dout, p.order[s] * p.sdo + i);
    st<T>(p.dweight, v * p.dim + i, sum * p.scale);
  }
}

template <typename F> void by_dtype(int dtype, F&& f) {
  if (dtype == MCPU_F32) f(float{});
  else if (dtype == MCPU_BF16) f(bf16{});
  else f(f16{});
}

}  // namespace

hipError_t embedding_fwd_launch(const EmbeddingParams& p, hipStream_t st) {
  by_dtype(p.dtype, [&](auto t) {
    hipLaunchKernelGGL(embedding_fwd_kernel<decltype(t)>, dim3(static_cast<unsigned>(p.tokens)), dim3(256), 0, st, p);
  });
  return hipGetLastError();
}

hipError_t embedding_bwd_launch(const EmbeddingParams& p, hipStream_t st) {
  // 256 ranges, one per CU, or more where a range would pass the table.
  int64_t range = (p.vocab + 255) / 256;
  if (range > kSortIds) range = kSortIds;
  hipLaunchKernelGGL(embedding_sort_kernel, dim3(static_cast<unsigned>((p.vocab + range - 1) / range)),
                     dim3(64 * kSortWaves), 0, st, p, static_cast<int>(range));
  by_dtype(p.dtype, [&](auto t) {
    hipLaunchKernelGGL(embedding_dw_kernel<decltype(t)>, dim3(static_cast<unsigned>((p.vocab + 3) / 4)), dim3(256), 0,
                       st, p);
  });
  return hipGetLastError();
}

}  // namespace mcpu
