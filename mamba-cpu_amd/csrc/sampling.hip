// Token sampling on gfx950, one workgroup per row of logits.
//
// Per row, with M the largest logit, T the temperature and w_i = exp((l_i - M) / T),
// in the order of the logits (descending, equal ones by index):
//   top-k  keeps the first k;
//   top-p  keeps a token while the mass before it, among the kept, is below
//          p times the mass of the kept;
//   min-p  keeps w_i >= min_p (w of the largest logit is 1);
//   the first token is always kept; the result is the kept token with the
//   largest w_i / noise_i, equal ones by index. With noise from Exp(1) that is
//   token i with probability w_i / sum of the kept (a race of exponentials).
// T <= 0 takes the first token. A row without a finite or infinite logit above
// -inf has no token: -1. NaN logits count as -inf.
//
// Every cut is a prefix of the order, so it is a pair: the key (the logit as an
// ordered integer) of its last token and the index up to which tokens of that
// key belong. The key is found by radix descent, 8 bits at a time, over counts
// or masses. Masses are added as integers (units of 2^-40 of the largest): the
// sums are exact in any order, so LDS atomics leave the result unchanged.
#include "lm_math.h"
#include "lm_params.h"

namespace mcpu {
namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr float kMassUnit = 1099511627776.0f;  // 2^40

// A logit as an unsigned integer of the same order; -0 and +0 are one key.
__device__ __forceinline__ uint32_t key_of(float l) {
  const uint32_t b = __builtin_bit_cast(uint32_t, l + 0.0f);
  return b ^ ((b >> 31) != 0 ? 0xffffffffu : 0x80000000u);
}

__device__ __forceinline__ uint64_t mass_of(float w) { return static_cast<uint64_t>(w * kMassUnit + 0.5f); }

struct Shared {
  uint32_t count[256];
  uint64_t mass[256];
  uint32_t u32[kWaves];
  uint64_t u64[kWaves];
  float f32[kWaves];
  uint32_t pick_key;
  uint64_t pick_above;
  uint32_t pick_count;
};

// The workgroup's maximum, in every thread. No barrier after the reads: the
// caller's next use of `slot` comes after another barrier.
__device__ __forceinline__ float group_max(float v, float* slot) {
  for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = v;
  __syncthreads();
  v = slot[0];
  for (int i = 1; i < kWaves; ++i) v = fmaxf(v, slot[i]);
  __syncthreads();
  return v;
}
__device__ __forceinline__ uint64_t group_sum(uint64_t v, uint64_t* slot) {
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0;
  for (int i = 0; i < kWaves; ++i) v += slot[i];
  __syncthreads();
  return v;
}
__device__ __forceinline__ uint32_t group_min(uint32_t v, uint32_t* slot) {
  for (int o = 32; o > 0; o >>= 1) v = min(v, __shfl_xor(v, o));
  if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = v;
  __syncthreads();
  v = slot[0];
  for (int i = 1; i < kWaves; ++i) v = min(v, slot[i]);
  __syncthreads();
  return v;
}

template <typename T> struct Row {
  const T* logits;
  int vocab;
  float top;  // the largest logit
  float temperature;

  __device__ __forceinline__ float at(int i) const {
    const float l = to_f32(logits[i]);
    return l == l ? l : -__builtin_inff();
  }
  // exp((l - M) / T); the largest logits, infinite ones too, weigh 1.
  __device__ __forceinline__ float weight(float l) const { return l == top ? 1.0f : exp_acc((l - top) / temperature); }
};

// A prefix of the order: keys above `key`, and of `key` the indices up to `last`.
struct Cut {
  uint32_t key, last;
  __device__ __forceinline__ bool has(uint32_t k, uint32_t i) const { return k > key || (k == key && i <= last); }
};

// The shortest prefix of `from` that holds `want` units: tokens (BY_MASS
// false) or mass, the last token counted if any of it is wanted. want >= 1 and
// at most what `from` holds.
template <bool BY_MASS, typename T>
__device__ Cut find_cut(const Row<T>& row, const Cut& from, uint64_t want, Shared& s) {
  uint32_t prefix = 0, above_bits = 0;  // the key's bits found so far, and their mask
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = threadIdx.x; i < 256; i += kThreads) {
      s.count[i] = 0;
      s.mass[i] = 0;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < row.vocab; i += kThreads) {
      const float l = row.at(i);
      const uint32_t k = key_of(l);
      if ((k & above_bits) != prefix || !from.has(k, i)) continue;
      const uint32_t bin = (k >> shift) & 255;
      if constexpr (BY_MASS) atomicAdd(reinterpret_cast<unsigned long long*>(&s.mass[bin]), mass_of(row.weight(l)));
      else atomicAdd(&s.count[bin], 1u);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      uint64_t left = want;
      int bin = 255;
      for (; bin > 0; --bin) {
        const uint64_t here = BY_MASS ? s.mass[bin] : s.count[bin];
        if (here >= left) break;
        left -= here;
      }
      s.pick_key = static_cast<uint32_t>(bin);
      s.pick_above = left;
    }
    __syncthreads();
    prefix |= s.pick_key << shift;
    above_bits |= 255u << shift;
    want = s.pick_above;
    __syncthreads();
  }
  // `want` units of the tokens with exactly this key, by index: how many tokens
  // that is, then where the last of them lies. A wave looks at a run of the row.
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int run = ((row.vocab + kWaves - 1) / kWaves + 63) / 64 * 64;
  const int t0 = w * run, t1 = min(t0 + run, row.vocab);
  uint32_t mine = 0;
  for (int i = t0 + lane; i - lane < t1; i += 64) {
    const float l = i < t1 ? row.at(i) : 0.f;
    const uint32_t k = key_of(l);
    mine += __popcll(__ballot(i < t1 && k == prefix && from.has(k, i)));
  }
  if (BY_MASS) {
    // All tokens of a key weigh the same.
    const float l = __builtin_bit_cast(float, prefix ^ ((prefix >> 31) != 0 ? 0x80000000u : 0xffffffffu));
    const uint64_t each = mass_of(row.weight(l));
    want = (want + each - 1) / each;  // the key's mass holds `want` >= 1, so each >= 1
  }
  if (lane == 0) s.u32[w] = mine;
  if (threadIdx.x == 0) s.pick_count = static_cast<uint32_t>(row.vocab - 1);
  __syncthreads();
  uint64_t seen = 0;
  for (int v = 0; v < w; ++v) seen += s.u32[v];
  if (seen < want && seen + mine >= want) {  // the wave that holds the last one
    for (int i = t0 + lane; i - lane < t1; i += 64) {
      const float l = i < t1 ? row.at(i) : 0.f;
      const uint32_t k = key_of(l);
      const uint64_t hit = __ballot(i < t1 && k == prefix && from.has(k, i));
      const uint32_t here = __popcll(hit);
      if (seen < want && seen + here >= want) {
        const uint32_t rank = static_cast<uint32_t>(want - seen);
        if (((hit >> lane) & 1) != 0 && __popcll(hit & ((1ull << lane) - 1)) + 1 == rank) s.pick_count = i;
      }
      seen += here;
    }
  }
  __syncthreads();
  const Cut cut{prefix, s.pick_count};
  __syncthreads();
  return cut;
}

template <typename T> __global__ __launch_bounds__(kThreads) void sample_kernel(const SampleParams p) {
  __shared__ Shared s;
  const int64_t r = blockIdx.x;
  Row<T> row;
  row.logits = static_cast<const T*>(p.logits) + r * p.sl;
  row.vocab = static_cast<int>(p.vocab);
  row.temperature = p.temperature_rows != nullptr ? p.temperature_rows[r] : p.temperature;
  const int64_t k = p.top_k_rows != nullptr ? p.top_k_rows[r] : p.top_k;
  const float top_p = p.top_p_rows != nullptr ? p.top_p_rows[r] : p.top_p;
  const float min_p = fminf(p.min_p_rows != nullptr ? p.min_p_rows[r] : p.min_p, 1.0f);

  float m = -__builtin_inff();
  for (int i = threadIdx.x; i < row.vocab; i += kThreads) m = fmaxf(m, row.at(i));
  row.top = group_max(m, s.f32);
  const bool none = row.top == -__builtin_inff();
  const bool greedy = !(row.temperature > 0.f);

  uint32_t best_i = 0xffffffffu;
  if (!none && greedy) {
    for (int i = threadIdx.x; i < row.vocab; i += kThreads)
      if (row.at(i) == row.top) best_i = min(best_i, static_cast<uint32_t>(i));
  } else if (!none) {
    Cut kept{0, static_cast<uint32_t>(row.vocab - 1)};
    if (k > 0 && k < row.vocab) kept = find_cut<false>(row, kept, static_cast<uint64_t>(k), s);
    if (top_p < 1.0f) {
      uint64_t total = 0;
      for (int i = threadIdx.x; i < row.vocab; i += kThreads) {
        const float l = row.at(i);
        if (kept.has(key_of(l), i)) total += mass_of(row.weight(l));
      }
      total = group_sum(total, s.u64);
      const double want = ceil(static_cast<double>(fmaxf(top_p, 0.f)) * static_cast<double>(total));
      kept = find_cut<true>(row, kept, want < 1.0 ? 1 : static_cast<uint64_t>(want), s);
    }
    const float* noise = p.noise + r * p.sn;
    float best = -1.0f;
    for (int i = threadIdx.x; i < row.vocab; i += kThreads) {
      const float l = row.at(i);
      if (!kept.has(key_of(l), i)) continue;
      const float w = row.weight(l);
      if (!(w >= min_p)) continue;
      const float score = w / fmaxf(noise[i], 1.17549435e-38f);
      if (score > best) {
        best = score;
        best_i = i;
      }
    }
    const float top = group_max(best, s.f32);
    if (best != top) best_i = 0xffffffffu;
  }
  best_i = group_min(best_i, s.u32);
  if (p.logprob != nullptr) {
    uint64_t total = 0;
    row.temperature = 1.0f;
    if (!none)
      for (int i = threadIdx.x; i < row.vocab; i += kThreads) total += mass_of(row.weight(row.at(i)));
    total = group_sum(total, s.u64);
    if (threadIdx.x == 0) {
      const float l = none ? 0.f : row.at(static_cast<int>(best_i));
      p.logprob[r] = none ? -__builtin_inff()
                          : (l == row.top ? 0.f : l - row.top) - logf(static_cast<float>(total) / kMassUnit);
    }
  }
  if (threadIdx.x == 0) p.token[r] = none ? -1 : static_cast<int64_t>(best_i);
}

}  // namespace

hipError_t sample_launch(const SampleParams& p, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>(p.rows)), block(kThreads);
  if (p.dtype == MCPU_F32) hipLaunchKernelGGL(sample_kernel<float>, grid, block, 0, st, p);
  else if (p.dtype == MCPU_BF16) hipLaunchKernelGGL(sample_kernel<bf16>, grid, block, 0, st, p);
  else hipLaunchKernelGGL(sample_kernel<f16>, grid, block, 0, st, p);
  return hipGetLastError();
}

}  // namespace mcpu
