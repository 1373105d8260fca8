// Token sampling on gfx950.
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
// T <= 0 takes the first token. A row without a logit above -inf has no token:
// -1. NaN logits count as -inf.
//
// Every cut is a prefix of the order, so it is a pair: the key (the logit as an
// ordered integer) of its last token and the index up to which tokens of that
// key belong. sample_row_kernel, one workgroup per row, reads the row once and
// keeps it in registers (up to kRowRegs logits per thread; longer rows are
// read again for every step), and finds the cuts in one of three ways:
//  - a short list: the k-th largest of the threads' maxima is at most the k-th
//    largest logit, so the logits from there up hold the first k and, for k up
//    to kListK, are few more. They are sorted in LDS; all that follows is a scan
//    over the list. Without top-k the kTryK-th maximum is tried: where the list
//    holds p of the mass it holds every token that top-p keeps.
//  - bins: counts or masses of kBins equal steps below M, and the sorted list of
//    the one bin that holds the cut.
//  - radix descent over the keys, 8 bits at a time, where a list overflows:
//    masses of equal logits, or a cut far below M.
// Masses are added as integers (units of 2^-40 of the largest): the sums are
// exact in any order, so LDS atomics leave the result unchanged. Where nothing
// is cut for any row, sample_slice_kernel takes rows in slices instead, so that
// few rows fill the chip, and sample_join_kernel compares their winners.
//
// The race runs on approximate scores first (v_exp_f32, v_rcp_f32: 8
// instructions a logit instead of 35); what comes within 2^-13 of the best is
// scored again with the division and exponential to the last place.
#include "lm_math.h"
#include "lm_params.h"

namespace mcpu {
namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr float kMassUnit = 1099511627776.0f;  // 2^40
constexpr float kNear = 1.0f - 0x1p-13f;
constexpr int kBins = 2048;
constexpr int kListK = 512;  // up to here the list holds about 1.4 k logits of its kThreads
constexpr int kTryK = 128;

// A logit as an unsigned integer of the same order; -0 and +0 are one key.
__device__ __forceinline__ uint32_t key_of(float l) {
  const uint32_t b = __builtin_bit_cast(uint32_t, l + 0.0f);
  return b ^ ((b >> 31) != 0 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __builtin_bit_cast(float, key ^ ((key >> 31) != 0 ? 0x80000000u : 0xffffffffu));
}

// w * 2^40 rounded down, from its two halves (w <= 1, so both are exact).
__device__ __forceinline__ uint64_t mass_of(float w) {
  const float hi = truncf(w * 256.0f);
  const float lo = (w * 256.0f - hi) * 4294967296.0f;
  return (static_cast<uint64_t>(static_cast<uint32_t>(hi)) << 32) | static_cast<uint32_t>(lo);
}

struct Shared {
  uint64_t bins[kBins];  // bins, and the radix descent's masses and counts
  uint64_t list[kThreads];
  float tops[kThreads];  // each thread's largest logit
  uint64_t u64[kWaves];
  uint32_t u32[kWaves];
  float f32[kWaves];
  uint32_t n, pick;
  uint64_t left;
};

// Reductions over the workgroup, in every thread, ending behind a barrier.
template <typename V, typename F> __device__ __forceinline__ V group_reduce(V v, V* slot, F&& join) {
  for (int o = 32; o > 0; o >>= 1) v = join(v, __shfl_xor(v, o));
  const int waves = blockDim.x >> 6;
  if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = v;
  __syncthreads();
  v = slot[0];
  for (int i = 1; i < waves; ++i) v = join(v, slot[i]);
  __syncthreads();
  return v;
}
__device__ __forceinline__ float group_max(float v, float* slot) {
  return group_reduce(v, slot, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float group_fsum(float v, float* slot) {
  return group_reduce(v, slot, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ uint64_t group_sum(uint64_t v, uint64_t* slot) {
  return group_reduce(v, slot, [](uint64_t a, uint64_t b) { return a + b; });
}
__device__ __forceinline__ uint32_t group_min(uint32_t v, uint32_t* slot) {
  return group_reduce(v, slot, [](uint32_t a, uint32_t b) { return min(a, b); });
}

// Sum over the threads before this one.
__device__ __forceinline__ uint64_t group_before(uint64_t v, uint64_t* slot) {
  const int lane = threadIdx.x & 63;
  uint64_t incl = v;
  for (int o = 1; o < 64; o <<= 1) {
    const uint64_t up = __shfl_up(incl, o);
    if (lane >= o) incl += up;
  }
  if (lane == 63) slot[threadIdx.x >> 6] = incl;
  __syncthreads();
  uint64_t before = incl - v;
  for (int i = 0; i < static_cast<int>(threadIdx.x >> 6); ++i) before += slot[i];
  __syncthreads();
  return before;
}

// ---- a row of logits ---------------------------------------------------------------------

typedef uint32_t u32x4_e2 __attribute__((ext_vector_type(4), aligned(2)));

template <typename T> constexpr uint32_t kLowest = std::is_same_v<T, bf16> ? 0xff80u : 0xfc00u;  // -inf, 16 bits

// kPer<T> neighbouring logits, 16 bytes, aligned to an element only.
template <typename T> constexpr int kPer = 16 / sizeof(T);
template <typename T> struct Pack {
  uint32_t w[4];
  __device__ __forceinline__ float at(int e) const {
    if constexpr (sizeof(T) == 4) return __builtin_bit_cast(float, w[e]);
    else return to_f32(__builtin_bit_cast(T, static_cast<uint16_t>(w[e / 2] >> (16 * (e % 2)))));
  }
};
// NaN counts as -inf.
__device__ __forceinline__ float clean(float l) { return l == l ? l : -__builtin_inff(); }
template <typename T> __device__ __forceinline__ Pack<T> clean(Pack<T> p) {
#pragma unroll
  for (int e = 0; e < kPer<T>; ++e) {
    const bool bad = !(p.at(e) == p.at(e));
    if constexpr (sizeof(T) == 4) p.w[e] = bad ? 0xff800000u : p.w[e];
    else if (e % 2 == 0) p.w[e / 2] = bad ? (p.w[e / 2] & 0xffff0000u) | kLowest<T> : p.w[e / 2];
    else p.w[e / 2] = bad ? (p.w[e / 2] & 0xffffu) | kLowest<T> << 16 : p.w[e / 2];
  }
  return p;
}

template <typename T> __device__ __forceinline__ Pack<T> load_pack(const T* row, int i, int vocab) {
  Pack<T> p;
  if (i + kPer<T> <= vocab) {
    const u32x4_e2 q = *reinterpret_cast<const u32x4_e2*>(row + i);
    p.w[0] = q.x;
    p.w[1] = q.y;
    p.w[2] = q.z;
    p.w[3] = q.w;
    return clean(p);
  }
  // The row's end: -inf beyond it.
  const uint32_t low = sizeof(T) == 4 ? 0xff800000u : kLowest<T> | kLowest<T> << 16;
  for (int e = 0; e < 4; ++e) p.w[e] = low;
  for (int e = 0; e < kPer<T>; ++e) {
    if (i + e >= vocab) break;
    if constexpr (sizeof(T) == 4) {
      p.w[e] = __builtin_bit_cast(uint32_t, row[i + e]);
    } else {
      const uint32_t b = __builtin_bit_cast(uint16_t, row[i + e]);
      p.w[e / 2] = e % 2 == 0 ? (p.w[e / 2] & 0xffff0000u) | b : (p.w[e / 2] & 0xffffu) | (b << 16);
    }
  }
  return clean(p);
}
// NP packs per thread in registers, or (NP = 0) the row read again for every use.
template <typename T, int NP> struct Row {
  const T* logits;
  int vocab;
  float top;          // the largest logit
  float ref, factor;  // weight_fast's: top (or the largest float), log2(e) / T
  float temperature;
  mutable Pack<T> pack[NP > 0 ? NP : 1];

  __device__ __forceinline__ float at(int i) const { return clean(to_f32(logits[i])); }
  __device__ __forceinline__ void load() {
    if constexpr (NP > 0)
#pragma unroll
      for (int j = 0; j < NP; ++j)
        pack[j] = load_pack(logits, min((j * kThreads + static_cast<int>(threadIdx.x)) * kPer<T>, vocab), vocab);
  }
  // f(index of the first, the pack) for each pack of this thread.
  template <typename F> __device__ __forceinline__ void each_pack(F&& f) const {
    if constexpr (NP > 0) {
      // The compiler is to forget what it knows of the values here: it would
      // keep every use's widened logits and comparisons for the next use, in
      // more registers than there are.
      int first = static_cast<int>(threadIdx.x) * kPer<T>;
      asm volatile("" : "+v"(first));
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        asm volatile("" : "+v"(pack[j].w[0]), "+v"(pack[j].w[1]), "+v"(pack[j].w[2]), "+v"(pack[j].w[3]));
        f(first + j * kThreads * kPer<T>, pack[j]);
      }
    } else {
      for (int i = threadIdx.x * kPer<T>; i < vocab; i += kThreads * kPer<T>) f(i, load_pack(logits, i, vocab));
    }
  }
  // f(index, logit); beyond the row's end the logit is -inf.
  template <typename F> __device__ __forceinline__ void each(F&& f) const {
    each_pack([&](int i, const Pack<T>& p) {
#pragma unroll
      for (int e = 0; e < kPer<T>; ++e) f(i + e, p.at(e));
    });
  }
  // exp((l - M) / T); the largest logits, infinite ones too, weigh 1.
  __device__ __forceinline__ float weight(float l) const { return l == top ? 1.0f : exp_acc((l - top) / temperature); }
  __device__ __forceinline__ float weight_fast(float l) const { return fast_exp2(fminf((l - ref) * factor, 0.f)); }
  __device__ __forceinline__ void set(float m, float t) {
    top = m;
    temperature = t;
    factor = kLog2e / t;
    ref = fminf(m, 3.402823466e38f);
  }
};

// A prefix of the order: keys above `key`, and of `key` the indices up to `last`.
struct Cut {
  uint32_t key, last;
  __device__ __forceinline__ bool has(uint32_t k, uint32_t i) const { return k > key || (k == key && i <= last); }
};

// The list's n <= kThreads entries (key << 32 | ~index) in descending order,
// thread t with entry t (0 behind the n-th): a bitonic network, whose steps
// within a wave are lane exchanges.
__device__ __forceinline__ uint64_t sorted_entry(Shared& s, int n) {
  const int t = threadIdx.x;
  uint64_t v = t < n ? s.list[t] : 0;
  for (int size = 2; size / 2 < n; size *= 2)
    for (int step = size / 2; step > 0; step /= 2) {
      uint64_t other;
      if (step < 64) {
        other = __shfl_xor(v, step);
      } else {
        __syncthreads();
        s.list[t] = v;
        __syncthreads();
        other = s.list[t ^ step];
      }
      const bool first = (t & step) == 0, down = (t & size) == 0;
      v = (v > other) == (first == down) ? v : other;
    }
  __syncthreads();
  return v;
}

// Appends what `in` accepts of the row to the list; how many that were, of
// which those beyond the list's end are lost.
template <typename R, typename F> __device__ __forceinline__ int collect(const R& row, Shared& s, F&& in) {
  if (threadIdx.x == 0) s.n = 0;
  __syncthreads();
  row.each([&](int i, float l) {
    if (i < row.vocab && in(i, l)) {
      const uint32_t at = atomicAdd(&s.n, 1u);
      if (at < kThreads) s.list[at] = (static_cast<uint64_t>(key_of(l)) << 32) | (0xffffffffu - i);
    }
  });
  __syncthreads();
  const int n = static_cast<int>(s.n);
  __syncthreads();
  return n;
}

// ---- cuts -----------------------------------------------------------------------------------

// The shortest prefix of `from` that holds `want` units: tokens (BY_MASS
// false) or mass, the last token counted if any of it is wanted; want >= 1 and
// at most what `from` holds. By radix descent over the keys.
template <bool BY_MASS, typename R> __device__ Cut radix_cut(const R& row, const Cut& from, uint64_t want, Shared& s) {
  uint32_t prefix = 0, mask = 0;  // the key's bits found so far, and which they are
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (threadIdx.x < 256) s.bins[threadIdx.x] = 0;
    __syncthreads();
    row.each([&](int i, float l) {
      const uint32_t k = key_of(l);
      if (i < row.vocab && (k & mask) == prefix && from.has(k, i))
        atomicAdd(reinterpret_cast<unsigned long long*>(&s.bins[(k >> shift) & 255]),
                  BY_MASS ? mass_of(row.weight_fast(l)) : 1ull);
    });
    __syncthreads();
    if (threadIdx.x == 0) {
      uint64_t left = want;
      int bin = 255;
      for (; bin > 0 && s.bins[bin] < left; --bin) left -= s.bins[bin];
      s.pick = static_cast<uint32_t>(bin);
      s.left = left;
    }
    __syncthreads();
    prefix |= s.pick << shift;
    mask |= 255u << shift;
    want = s.left;
    __syncthreads();
  }
  // `want` units of the tokens with exactly this key, by index: how many tokens
  // that is (they weigh the same), then where the last of them lies. A wave
  // looks at a run of the row.
  if (BY_MASS) {
    const uint64_t each = mass_of(row.weight_fast(value_of(prefix)));
    want = (want + each - 1) / each;  // the key's mass holds `want` >= 1, so each >= 1
  }
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int run = ((row.vocab + kWaves - 1) / kWaves + 63) / 64 * 64;
  const int t0 = w * run, t1 = min(t0 + run, row.vocab);
  auto hits = [&](int i) {
    const uint32_t k = key_of(i < t1 ? row.at(i) : 0.f);
    return __ballot(i < t1 && k == prefix && from.has(k, i));
  };
  uint32_t mine = 0;
  for (int i = t0 + lane; i - lane < t1; i += 64) mine += __popcll(hits(i));
  if (lane == 0) s.u32[w] = mine;
  if (threadIdx.x == 0) s.pick = static_cast<uint32_t>(row.vocab - 1);
  __syncthreads();
  uint64_t seen = 0;
  for (int v = 0; v < w; ++v) seen += s.u32[v];
  if (seen < want && seen + mine >= want) {  // the wave that holds the last one
    for (int i = t0 + lane; i - lane < t1; i += 64) {
      const uint64_t hit = hits(i);
      const uint32_t here = __popcll(hit);
      if (seen < want && seen + here >= want && ((hit >> lane) & 1) != 0 &&
          __popcll(hit & ((1ull << lane) - 1)) + 1 == want - seen)
        s.pick = i;
      seen += here;
    }
  }
  __syncthreads();
  const Cut cut{prefix, s.pick};
  __syncthreads();
  return cut;
}

// The same by bins of equal width below M: as far as the row reaches, at most
// 24 T (where w is 4e-11); the last bin takes what lies beyond.
template <bool BY_MASS, typename R>
__device__ __forceinline__ Cut find_cut(const R& row, float low, const Cut& from, uint64_t want, Shared& s) {
  const float scale = (kBins - 1) / fmaxf(fminf(24.0f * row.temperature, row.top - low), 1e-30f);
  auto bin_of = [&](float l) { return static_cast<int>(fmaxf(fminf((row.ref - l) * scale, kBins - 1.0f), 0.f)); };
  for (int i = threadIdx.x; i < kBins; i += kThreads) s.bins[i] = 0;
  __syncthreads();
  row.each([&](int i, float l) {
    if (i < row.vocab && from.has(key_of(l), i))
      atomicAdd(reinterpret_cast<unsigned long long*>(&s.bins[bin_of(l)]),
                BY_MASS ? mass_of(row.weight_fast(l)) : 1ull);
  });
  __syncthreads();
  const uint64_t b0 = s.bins[2 * threadIdx.x], b1 = s.bins[2 * threadIdx.x + 1];
  const uint64_t before = group_before(b0 + b1, s.u64);
  if (threadIdx.x == 0) s.pick = kBins - 1;  // rounding may leave the sum short of `want`
  __syncthreads();
  if (before < want && before + b0 + b1 >= want) {
    const bool second = before + b0 < want;
    s.pick = 2 * threadIdx.x + second;
    s.left = want - before - (second ? b0 : 0);
  }
  __syncthreads();
  const int bin = static_cast<int>(s.pick);
  const uint64_t left = s.left;
  __syncthreads();
  if (bin < kBins - 1) {
    const int n = collect(row, s, [&](int i, float l) { return from.has(key_of(l), i) && bin_of(l) == bin; });
    if (n <= kThreads) {
      const uint64_t e = sorted_entry(s, n);
      const bool in = static_cast<int>(threadIdx.x) < n;
      const uint64_t unit = in ? (BY_MASS ? mass_of(row.weight_fast(value_of(e >> 32))) : 1) : 0;
      const uint64_t at = group_before(unit, s.u64);
      if (in && at < left && at + unit >= left) s.left = e;
      __syncthreads();
      const Cut cut{static_cast<uint32_t>(s.left >> 32), 0xffffffffu - static_cast<uint32_t>(s.left)};
      __syncthreads();
      return cut;
    }
  }
  return radix_cut<BY_MASS>(row, from, want, s);
}

// The largest key of the threads' maxima that at least `want` of them reach,
// or one a little lower: bisection, by every wave for itself.
__device__ __forceinline__ uint32_t maxima_key(const Shared& s, int want) {
  uint32_t k[kThreads / 64];
#pragma unroll
  for (int j = 0; j < kThreads / 64; ++j) k[j] = key_of(s.tops[j * 64 + (threadIdx.x & 63)]);
  uint32_t lo = 0, hi = 0xffffffffu;  // all reach lo; fewer than `want` reach hi
  while (hi - lo > 1) {
    const uint32_t mid = lo + (hi - lo) / 2;
    int n = 0;
#pragma unroll
    for (int j = 0; j < kThreads / 64; ++j) n += __popcll(__ballot(k[j] >= mid));
    if (n < want) {
      hi = mid;
    } else {
      lo = mid;
      if (n <= want + want / 4 + 8) break;
    }
  }
  return lo;
}

// ---- the race ----------------------------------------------------------------------------------

__device__ __forceinline__ float noise_at(const float* noise, int i) { return fmaxf(noise[i], 1.17549435e-38f); }

// The workgroup's largest score and, of those who hold it, the lowest index.
__device__ __forceinline__ uint32_t winner(float score, uint32_t i, float* f32, uint32_t* u32) {
  const float top = group_max(score, f32);
  return group_min(score == top ? i : 0xffffffffu, u32);
}

template <typename T, int NP> __global__ __launch_bounds__(kThreads) void sample_row_kernel(const SampleParams p) {
  __shared__ Shared s;
  const int64_t r = blockIdx.x;
  Row<T, NP> row;
  row.logits = static_cast<const T*>(p.logits) + r * p.sl;
  row.vocab = static_cast<int>(p.vocab);
  // An infinite temperature would weigh -inf logits too (0 x inf).
  float temperature = p.temperature_rows != nullptr ? p.temperature_rows[r] : p.temperature;
  if (temperature > 1e30f) temperature = 1e30f;
  int k = p.top_k_rows != nullptr ? p.top_k_rows[r] : p.top_k;
  const float top_p = p.top_p_rows != nullptr ? p.top_p_rows[r] : p.top_p;
  const float min_p = fminf(p.min_p_rows != nullptr ? p.min_p_rows[r] : p.min_p, 1.0f);
  if (k >= row.vocab) k = 0;
  row.load();

  const float inf = __builtin_inff();
  float m = -inf, low = inf;
  row.each([&](int, float l) {
    m = fmaxf(m, l);
    low = fminf(low, l == -inf ? inf : l);
  });
  s.tops[threadIdx.x] = m;
  m = group_max(m, s.f32);
  if (m == -inf) {
    if (threadIdx.x == 0) {
      p.token[r] = -1;
      if (p.logprob != nullptr) p.logprob[r] = -inf;
    }
    return;
  }
  const bool greedy = !(temperature > 0.f);
  float total1 = 0.f;  // sum of exp(l - M), for the log-probability
  row.set(m, 1.0f);
  if (p.logprob != nullptr) {
    row.each([&](int, float l) { total1 += row.weight_fast(l); });
    total1 = group_fsum(total1, s.f32);
  }

  uint32_t token = 0xffffffffu;
  if (greedy) {
    row.each([&](int i, float l) {
      if (l == m) token = min(token, static_cast<uint32_t>(i));
    });
    token = group_min(token, s.u32);
  } else {
    row.set(m, temperature);
    const float* noise = p.noise + r * p.sn;
    const bool few = k > 0 && k <= kListK;
    float total = 0.f;  // mass of all, where top-p is asked without top-k
    if (top_p < 1.0f && k == 0) {
      if (temperature == 1.0f && p.logprob != nullptr) {
        total = total1;
      } else {
        row.each([&](int, float l) { total += row.weight_fast(l); });
        total = group_fsum(total, s.f32);
      }
    }
    const float part = fmaxf(top_p, 0.f);
    if (few || (top_p < 1.0f && k == 0)) {
      // The short list.
      const float from = row.vocab <= kThreads ? -inf : value_of(maxima_key(s, few ? k : kTryK));
      const int n = collect(row, s, [&](int, float l) { return l >= from; });
      if (n <= kThreads) {
        const bool in = static_cast<int>(threadIdx.x) < n;
        bool holds = few;
        if (!few) {
          const uint64_t e = in ? s.list[threadIdx.x] : 0;
          holds = row.vocab <= kThreads ||
                  static_cast<float>(group_sum(in ? mass_of(row.weight(value_of(e >> 32))) : 0, s.u64)) >
                      part * total * kMassUnit * kNear;
        }
        if (holds) {
          const uint64_t e = sorted_entry(s, n);
          const float w = in ? row.weight(value_of(e >> 32)) : 0.f;
          const uint32_t i = 0xffffffffu - static_cast<uint32_t>(e);
          bool keep = in && (!few || static_cast<int>(threadIdx.x) < k);
          if (top_p < 1.0f) {
            const uint64_t mass = keep ? mass_of(w) : 0;
            const uint64_t all = few ? group_sum(mass, s.u64) : static_cast<uint64_t>(total * kMassUnit);
            const double want = ceil(static_cast<double>(part) * static_cast<double>(all));
            keep = group_before(mass, s.u64) < static_cast<uint64_t>(want) && keep;
          }
          keep = (keep && w >= min_p) || threadIdx.x == 0;
          token = winner(keep ? w / noise_at(noise, static_cast<int>(i)) : -1.0f, i, s.f32, s.u32);
        }
      }
    }
    if (token == 0xffffffffu) {
      Cut kept{key_of(-inf), static_cast<uint32_t>(row.vocab - 1)};  // everything
      low = -group_max(-low, s.f32);
      if (k > 0) {
        kept = find_cut<false>(row, low, kept, static_cast<uint64_t>(k), s);
        if (top_p < 1.0f) {
          row.each([&](int i, float l) { total += i < row.vocab && kept.has(key_of(l), i) ? row.weight_fast(l) : 0.f; });
          total = group_fsum(total, s.f32);
        }
      }
      if (top_p < 1.0f) {
        const double want = ceil(static_cast<double>(part) * static_cast<double>(total) * kMassUnit);
        kept = find_cut<true>(row, low, kept, want < 1.0 ? 1 : static_cast<uint64_t>(want), s);
      }
      // The race over the row. `edge` is the cut's logit.
      const float edge = value_of(kept.key);
      auto scores = [&](auto&& f) {
        row.each_pack([&](int i, const Pack<T>& q) {
          bool any = false;
          float l[kPer<T>];
          bool in[kPer<T>];
#pragma unroll
          for (int e = 0; e < kPer<T>; ++e) {
            l[e] = q.at(e);
            in[e] = l[e] > edge || (l[e] == edge && static_cast<uint32_t>(i + e) <= kept.last);
            if (in[e] && min_p > 0.f) {
              const float w = row.weight_fast(l[e]);
              in[e] = w >= min_p * (2.0f - kNear) || (w >= min_p * kNear && row.weight(l[e]) >= min_p);
            }
            any |= in[e];
          }
          if (!any) return;
          if (i + kPer<T> <= row.vocab) {
#pragma unroll
            for (int h = 0; h < kPer<T>; h += 4) {
              float q4[4];
              ld4_elem<float>(noise, i + h, q4);
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (in[h + e]) f(i + h + e, l[h + e], fmaxf(q4[e], 1.17549435e-38f));
            }
          } else {
#pragma unroll
            for (int e = 0; e < kPer<T>; ++e)
              if (in[e] && i + e < row.vocab) f(i + e, l[e], noise_at(noise, i + e));
          }
        });
      };
      float best = -1.0f;
      scores([&](int, float l, float q) { best = fmaxf(best, row.weight_fast(l) * fast_rcp(q)); });
      const float bar = group_max(best, s.f32) * kNear;
      float score = -1.0f;
      uint32_t at = 0xffffffffu;
      if (best >= bar) {
        scores([&](int i, float l, float q) {
          if (row.weight_fast(l) * fast_rcp(q) < bar) return;
          const float exact = row.weight(l) / q;
          if (exact > score) {
            score = exact;
            at = static_cast<uint32_t>(i);
          }
        });
      }
      token = winner(score, at, s.f32, s.u32);
    }
  }
  if (threadIdx.x == 0) {
    p.token[r] = static_cast<int64_t>(token);
    if (p.logprob != nullptr && token < static_cast<uint32_t>(row.vocab)) {
      const float l = row.at(static_cast<int>(token));
      p.logprob[r] = (l == m ? 0.f : l - m) - logf(total1);
    }
  }
}

}  // namespace

hipError_t sample_launch(const SampleParams& p, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>(p.rows)), block(kThreads);
  auto by_size = [&](auto t) {
    using T = decltype(t);
    constexpr int kFull = 64 / kPer<T>, kSmall = 16 / kPer<T>;  // packs of 64 and 16 logits per thread
    if (p.vocab <= 16 * kThreads) hipLaunchKernelGGL((sample_row_kernel<T, kSmall>), grid, block, 0, st, p);
    else if (p.vocab <= 64 * kThreads) hipLaunchKernelGGL((sample_row_kernel<T, kFull>), grid, block, 0, st, p);
    else hipLaunchKernelGGL((sample_row_kernel<T, 0>), grid, block, 0, st, p);
  };
  if (p.dtype == MCPU_F32) by_size(float{});
  else if (p.dtype == MCPU_BF16) by_size(bf16{});
  else by_size(f16{});
  return hipGetLastError();
}

}  // namespace mcpu
