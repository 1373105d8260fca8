// Embedding on gfx950: out_t = scale weight[id_t], and its gradient
// dweight_v = scale sum_{t: id_t = v} dout_t.
//
// The gradient is a segmented sum over the tokens sorted by id: the sum of an
// id runs over its tokens in a fixed order, in float32, and is rounded once, so
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

// One wave per token, four elements per lane.
template <typename T> __global__ __launch_bounds__(256) void embedding_fwd_kernel(const EmbeddingParams p) {
  const int lane = threadIdx.x & 63;
  const int64_t t = blockIdx.x * 4ll + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (t >= p.tokens) return;
  const int64_t id = id_at(p, t);
  const bool in = id >= 0 && id < p.vocab;
  const T* from = static_cast<const T*>(p.weight) + (in ? id : 0) * p.sw;
  T* to = static_cast<T*>(p.out) + t * p.dim;
  for (int64_t i = lane * 4; i < p.dim; i += 256) {
    const int n = upto4(p.dim - i);
    float v[4] = {};
    if (in) ld_upto4<T>(from, i, n, v);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] *= p.scale;
    st_upto4<T>(to, i, n, v);
  }
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

// Adds the rows of dout at the sorted positions [s0, s1), at most 64, element
// i to i + n: the positions are read at once, one per lane, and passed on as
// scalars, so that the rows' loads do not wait for each other.
template <typename T>
__device__ __forceinline__ void add_rows(const EmbeddingParams& p, int mine, int s0, int s1, int64_t i, int n,
                                         float (&sum)[4]) {
  const T* dout = static_cast<const T*>(p.dout);
  int s = s0;
  for (; s + 4 <= s1; s += 4) {
    float v[4][4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int64_t t = __builtin_amdgcn_readlane(mine, s + k - s0);
      ld_upto4<T>(dout + t * p.sdo, i, n, v[k]);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] += v[k][e];
  }
  for (; s < s1; ++s) {
    const int64_t t = __builtin_amdgcn_readlane(mine, s - s0);
    float v[4];
    ld_upto4<T>(dout + t * p.sdo, i, n, v);
#pragma unroll
    for (int e = 0; e < 4; ++e) sum[e] += v[e];
  }
}

// dweight, in one launch of two kinds of workgroups. The first `chunks` take
// kEmbedChunk sorted positions each and add, per id with more tokens than that
// (a hot id), the part of its rows that lies here: the part of the id at the
// chunk's first position goes to slot 0, that of a hot id starting later to
// slot 1 (it runs past the chunk's end, so there is at most one). The others
// give each wave a row of dweight: the sum of an id with few tokens, or zeros.
// Hot rows are joined by embedding_join_kernel. Without this split one wave
// adds the most frequent id alone: 3.5 ms of 16384 tokens' 5.1 ms.
template <typename T>
__global__ __launch_bounds__(256) void embedding_dw_kernel(const EmbeddingParams p, int chunks) {
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (static_cast<int>(blockIdx.x) < chunks) {
    const int c0 = blockIdx.x * kEmbedChunk, valid = p.start[p.vocab];
    const int c1 = min(c0 + kEmbedChunk, valid);
    int s = c0;
    while (s < c1) {
      const int64_t id = id_at(p, p.order[s]);
      const int end = p.start[id + 1];
      if (end - p.start[id] > kEmbedChunk) {
        const int s1 = min(end, c1), slot = s == c0 ? 0 : 1;
        const int mine = lane < s1 - s ? p.order[s + lane] : 0;
        float* part = p.part + (blockIdx.x * 2ll + slot) * p.dim;
        for (int64_t i = (w * 64 + lane) * 4; i < p.dim; i += 1024) {
          const int n = upto4(p.dim - i);
          float sum[4] = {};
          add_rows<T>(p, mine, s, s1, i, n, sum);
          st_upto4<float>(part, i, n, sum);
        }
      }
      s = end;
    }
    return;
  }
  const int64_t v = (blockIdx.x - chunks) * 4ll + w;
  if (v >= p.vocab) return;
  const int s0 = p.start[v], s1 = p.start[v + 1];
  if (s1 - s0 > kEmbedChunk) return;
  const int mine = lane < s1 - s0 ? p.order[s0 + lane] : 0;
  T* row = static_cast<T*>(p.dweight) + v * p.dim;
  for (int64_t i = lane * 4; i < p.dim; i += 256) {
    const int n = upto4(p.dim - i);
    float sum[4] = {};
    add_rows<T>(p, mine, s0, s1, i, n, sum);
#pragma unroll
    for (int e = 0; e < 4; ++e) sum[e] *= p.scale;
    st_upto4<T>(row, i, n, sum);
  }
}

constexpr int kJoinWaves = 16;

// The row of a hot id, by the workgroups of the chunk it starts in (256
// elements each): its parts in every kJoinWaves-th chunk are added by one wave
// each, then the waves' sums in order.
template <typename T>
__global__ __launch_bounds__(64 * kJoinWaves) void embedding_join_kernel(const EmbeddingParams p) {
  __shared__ float sums[kJoinWaves][256];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c0 = blockIdx.x * kEmbedChunk, valid = p.start[p.vocab];
  if (c0 >= valid) return;
  // The hot id that starts here is the last one of the chunk: every other id
  // that starts here ends here.
  const int64_t id = id_at(p, p.order[min(c0 + kEmbedChunk, valid) - 1]);
  const int first = p.start[id], end = p.start[id + 1];
  if (end - first <= kEmbedChunk || first < c0) return;
  const int last = (end - 1) / kEmbedChunk;
  const int64_t i = blockIdx.y * 256ll + lane * 4;
  const int n = i < p.dim ? upto4(p.dim - i) : 0;
  float sum[4] = {};
  if (n > 0) {
#pragma unroll 4
    for (int64_t c = static_cast<int64_t>(blockIdx.x) + w; c <= last; c += kJoinWaves) {
      const int slot = c == blockIdx.x && first > c0 ? 1 : 0;
      float v[4];
      ld_upto4<float>(p.part + (c * 2 + slot) * p.dim, i, n, v);
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] += v[e];
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) sums[w][lane * 4 + e] = sum[e];
  __syncthreads();
  const int64_t col = blockIdx.y * 256ll + threadIdx.x;
  if (threadIdx.x < 256 && col < p.dim) {
    float total = 0.f;
    for (int v = 0; v < kJoinWaves; ++v) total += sums[v][threadIdx.x];
    st<T>(p.dweight, id * p.dim + col, total * p.scale);
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
    hipLaunchKernelGGL(embedding_fwd_kernel<decltype(t)>, dim3(static_cast<unsigned>((p.tokens + 3) / 4)), dim3(256),
                       0, st, p);
  });
  return hipGetLastError();
}

// Chunks of sorted positions, or none where no id can be hot.
int64_t embedding_chunks(int64_t tokens) {
  return tokens > kEmbedChunk ? (tokens + kEmbedChunk - 1) / kEmbedChunk : 0;
}

hipError_t embedding_bwd_launch(const EmbeddingParams& p, hipStream_t st) {
  // 256 ranges, one per CU, or more where a range would pass the table.
  int64_t range = (p.vocab + 255) / 256;
  if (range > kSortIds) range = kSortIds;
  hipLaunchKernelGGL(embedding_sort_kernel, dim3(static_cast<unsigned>((p.vocab + range - 1) / range)),
                     dim3(64 * kSortWaves), 0, st, p, static_cast<int>(range));
  const int chunks = static_cast<int>(embedding_chunks(p.tokens));
  by_dtype(p.dtype, [&](auto t) {
    using T = decltype(t);
    hipLaunchKernelGGL(embedding_dw_kernel<T>, dim3(static_cast<unsigned>(chunks + (p.vocab + 3) / 4)), dim3(256), 0,
                       st, p, chunks);
    if (chunks > 0)
      hipLaunchKernelGGL(embedding_join_kernel<T>, dim3(chunks, static_cast<unsigned>((p.dim + 255) / 256)),
                         dim3(64 * kJoinWaves), 0, st, p);
  });
  return hipGetLastError();
}

}  // namespace mcpu
