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
// key belong. sample_row_kernel, one workgroup per row, finds the cuts in one of
// three ways:
//  - a short list: the k-th largest of the threads' maxima is at most the k-th
//    largest logit, so the logits from there up hold the first k and, for k up
//    to kListK, are few more. They are sorted in LDS; all that follows is a scan
//    over the list. Without top-k the kTryK-th maximum is tried: where the list
//    holds p of the mass it holds every token that top-p keeps. Min-p's own
//    lowest logit, M + T log(min_p), does as well.
//  - bins: counts or masses of kBins equal steps below M, and the sorted list of
//    the one bin that holds the cut.
//  - radix descent over the keys, 8 bits at a time, where a list overflows:
//    masses of equal logits, or a cut far below M.
// Masses are added as integers: the sums are exact in any order, so LDS atomics
// leave the result unchanged. Bins count in units of 2^-31 of the total, each
// logit to the nearest: the cut is off by at most vocab / 2 units, which is allowed
// up to 1/16 of what top-p cuts off (and 2^-13 of the total). Beyond that, for
// top-p near 1, and in the radix descent, masses have 64 bits. Where
// nothing is cut for any row, sample_slice_kernel takes rows in slices instead,
// so that few rows fill the chip, and sample_join_kernel compares their winners.
//
// The race runs on approximate logarithms of the scores first, 9 instructions a
// logit, of which a pack's largest is kept; what comes near the best is scored
// again with the division and exponential to the last place. A pass over a row
// is bound by its instructions on one CU: 50280 logits take 0.35 us for each. So
// NaN are cleaned only in rows that have any, and what few logits need is worked
// off in loops over bits.
#include "launch.h"
#include "lm_math.h"
#include "lm_params.h"

namespace mcpu {
namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
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

struct Shared {
  union {
    uint32_t bins[kBins];
    uint64_t wide_bins[kBins];  // the radix descent's, too
  };
  uint64_t list[kThreads];
  float tops[kThreads];  // each thread's largest logit
  uint32_t u32[kWaves];
  float f32[kWaves];
  uint32_t odd[kWaves];
  uint32_t n, pick;
  uint64_t left, entry;
};

// Reductions over the WAVES waves of a workgroup, in every thread, ending
// behind a barrier.
template <int WAVES, typename V, typename F> __device__ __forceinline__ V group_reduce(V v, V* slot, F&& join) {
  for (int o = 32; o > 0; o >>= 1) v = join(v, __shfl_xor(v, o));
  if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = v;
  __syncthreads();
  V each[WAVES];
#pragma unroll
  for (int i = 0; i < WAVES; ++i) each[i] = slot[i];
  v = each[0];
#pragma unroll
  for (int i = 1; i < WAVES; ++i) v = join(v, each[i]);
  __syncthreads();
  return v;
}
template <int WAVES = kWaves> __device__ __forceinline__ float group_max(float v, float* slot) {
  return group_reduce<WAVES>(v, slot, [](float a, float b) { return fmaxf(a, b); });
}
template <int WAVES = kWaves> __device__ __forceinline__ float group_fsum(float v, float* slot) {
  return group_reduce<WAVES>(v, slot, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ uint32_t group_usum(uint32_t v, uint32_t* slot) {
  return group_reduce<kWaves>(v, slot, [](uint32_t a, uint32_t b) { return a + b; });
}
template <int WAVES = kWaves> __device__ __forceinline__ uint32_t group_min(uint32_t v, uint32_t* slot) {
  return group_reduce<WAVES>(v, slot, [](uint32_t a, uint32_t b) { return min(a, b); });
}

// Sum over the threads before this one.
template <typename V> __device__ __forceinline__ V group_before(V v, V* slot) {
  const int lane = threadIdx.x & 63;
  V incl = v;
  for (int o = 1; o < 64; o <<= 1) {
    const V up = __shfl_up(incl, o);
    if (lane >= o) incl += up;
  }
  if (lane == 63) slot[threadIdx.x >> 6] = incl;
  __syncthreads();
  V each[kWaves], before = incl - v;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) each[i] = slot[i];
#pragma unroll
  for (int i = 0; i < kWaves; ++i) before += i < static_cast<int>(threadIdx.x >> 6) ? each[i] : 0;
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
  // The same for an e that is not a constant.
  __device__ __forceinline__ float pick(int e) const {
    const int j = sizeof(T) == 4 ? e : e / 2;
    const uint32_t w0 = w[0], w1 = w[1], w2 = w[2], w3 = w[3];
    const uint32_t word = j < 2 ? (j == 0 ? w0 : w1) : (j == 2 ? w2 : w3);
    if constexpr (sizeof(T) == 4) return __builtin_bit_cast(float, word);
    else return to_f32(__builtin_bit_cast(T, static_cast<uint16_t>(word >> (16 * (e % 2)))));
  }
  // Bit e: whether f holds for element e. For what is rare: the bits are then
  // worked off in a loop, where code for each element would crowd out the passes.
  template <typename F> __device__ __forceinline__ uint32_t which(F&& f) const {
    uint32_t hits = 0;
#pragma unroll
    for (int e = 0; e < kPer<T>; ++e) hits |= f(at(e)) ? 1u << e : 0u;
    return hits;
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
    return p;
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
  return p;
}
// x cut to [0, 1].
__device__ __forceinline__ float upto1(float x) { return __builtin_amdgcn_fmed3f(x, 0.f, 1.f); }

// A row, read again from the cache for every use: it is there (32 rows of 50280
// bf16 logits fill 3.2 of the 4 MB of an XCD's L2), and holding 50 logits a
// thread in registers spilled (35 against 27 us for one float32 row).
template <typename T> struct Row {
  static constexpr int kE = kPer<T>;
  const T* logits;
  int vocab;
  bool odd;           // there are NaN in it
  float top;          // the largest logit
  float ref, factor;  // weight_fast's: top (or the largest float), log2(e) / T
  float temperature;

  __device__ __forceinline__ float at(int i) const { return clean(to_f32(logits[i])); }
  // f(index of the first, the pack) for each pack of this thread, kAhead packs
  // on their way at once.
  template <typename F> __device__ __forceinline__ void each_pack(F&& f) const {
    constexpr int kAhead = 4;
    for (int i0 = threadIdx.x * kPer<T>; i0 < vocab; i0 += kAhead * kThreads * kPer<T>) {
      Pack<T> p[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) p[j] = load_pack(logits, i0 + j * kThreads * kPer<T>, vocab);
      if (odd) {
#pragma unroll
        for (int j = 0; j < kAhead; ++j) p[j] = clean(p[j]);
      }
#pragma unroll
      for (int j = 0; j < kAhead; ++j)
        if (i0 + j * kThreads * kPer<T> < vocab) f(i0 + j * kThreads * kPer<T>, p[j]);
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
  // Clamped to 1, for M = inf (a modifier of v_exp_f32, without an instruction).
  __device__ __forceinline__ float weight_fast(float l) const { return upto1(fast_exp2(steps(l))); }
  // log2 of the weight; of an infinite M itself infinity.
  __device__ __forceinline__ float steps(float l) const { return (l - ref) * factor; }
  // Temperatures beyond 1e-30 and 1e30 act as those (log2(e) / T stays a number,
  // also times 0 and infinity).
  __device__ __forceinline__ void set(float m, float t) {
    top = m;
    temperature = __builtin_amdgcn_fmed3f(t, 1e-30f, 1e30f);
    factor = kLog2e / temperature;
    ref = fminf(m, 3.402823466e38f);
  }
};

// A prefix of the order: logits above `edge`, and of `edge` the indices up to `last`.
struct Cut {
  float edge;
  uint32_t last;
  // Not what lies beyond the row's end: it is -inf, and `last` lies in the row.
  __device__ __forceinline__ bool has(float l, int i) const {
    return l > edge || (l == edge && static_cast<uint32_t>(i) <= last);
  }
};

// The value of lane ^ STEP, by DPP moves: xor 4 is half a row mirrored (xor 7)
// and quads reversed (xor 3), xor 8 a row turned by half.
template <int STEP> __device__ __forceinline__ uint64_t lane_xor(uint64_t v) {
  auto half = [](int x) {
    constexpr int kRowRor8 = 0x128;
    if constexpr (STEP == 1) return __builtin_amdgcn_mov_dpp(x, kQuadXor1, 0xf, 0xf, true);
    else if constexpr (STEP == 2) return __builtin_amdgcn_mov_dpp(x, kQuadXor2, 0xf, 0xf, true);
    else if constexpr (STEP == 4)
      return __builtin_amdgcn_mov_dpp(__builtin_amdgcn_mov_dpp(x, kQuadXor3, 0xf, 0xf, true), kRowHalfMirror, 0xf, 0xf,
                                      true);
    else return __builtin_amdgcn_mov_dpp(x, kRowRor8, 0xf, 0xf, true);
  };
  const uint32_t lo = half(static_cast<int>(v)), hi = half(static_cast<int>(v >> 32));
  return static_cast<uint64_t>(hi) << 32 | lo;
}

// The list's n <= kThreads entries (key << 32 | ~index) in descending order,
// thread t with entry t (0 behind the n-th). Short lists by counting, for each
// entry, those above it (all are different); longer ones by a bitonic network,
// whose steps within a wave are lane exchanges. 55 entries take 0.6 us against
// 3 by the network, which wins from about 300 on (700: 8 us).
__device__ __forceinline__ uint64_t sorted_entry(Shared& s, int n) {
  const int t = threadIdx.x;
  uint64_t v = t < n ? s.list[t] : 0;
  if (n <= 256) {
    if (t >= n && t < (n + 7) / 8 * 8) s.list[t] = 0;
    __syncthreads();
    int rank = 0;
    if ((t & ~63) < n)
      for (int i = 0; i < n; i += 8)
#pragma unroll
        for (int j = 0; j < 8; ++j) rank += s.list[i + j] > v;
    __syncthreads();
    if (t < n) s.list[rank] = v;
    __syncthreads();
    v = t < n ? s.list[t] : 0;
    __syncthreads();
    return v;
  }
  for (int size = 2; size / 2 < n; size *= 2) {
    auto keep = [&](uint64_t other, int step) {
      const bool first = (t & step) == 0, down = (t & size) == 0;
      v = (v > other) == (first == down) ? v : other;
    };
    for (int step = size / 2; step >= 64; step /= 2) {
      __syncthreads();
      s.list[t] = v;
      __syncthreads();
      keep(s.list[t ^ step], step);
    }
    for (int step = min(size / 2, 32); step >= 16; step /= 2) keep(__shfl_xor(v, step), step);
    if (size > 8) keep(lane_xor<8>(v), 8);
    if (size > 4) keep(lane_xor<4>(v), 4);
    if (size > 2) keep(lane_xor<2>(v), 2);
    keep(lane_xor<1>(v), 1);
  }
  __syncthreads();
  return v;
}

// Appends a logit to the list; what comes behind the list's end is only counted.
__device__ __forceinline__ void append(Shared& s, float l, int i) {
  const uint32_t at = atomicAdd(&s.n, 1u);
  if (at < kThreads) s.list[at] = (static_cast<uint64_t>(key_of(l)) << 32) | (0xffffffffu - i);
}

// ---- cuts -----------------------------------------------------------------------------------

// What a logit counts for a cut: one token, or its mass, `unit` to a weight of 1.
template <bool BY_MASS, typename U, typename R>
__device__ __forceinline__ U units(const R& row, float l, float unit) {
  return BY_MASS ? static_cast<U>(fmaf(row.weight_fast(l), unit, 0.5f)) : U{1};
}
// The unit of 64-bit masses: 2^(62 - bits of vocab), so that a row's sum fits 63 bits.
template <typename R> __device__ __forceinline__ float wide_unit(const R& row) {
  return ldexpf(1.0f, 30 + __builtin_clz(row.vocab));
}
// The fraction `part` of a mass: at least 1 unit, and not more than there is.
__device__ __forceinline__ uint64_t fraction(float part, uint64_t all) {
  const double want = ceil(static_cast<double>(part) * static_cast<double>(all));
  return want < 1.0 ? 1 : min(static_cast<uint64_t>(want), all);
}

// The shortest prefix of `from` that holds what is wanted, the last token
// counted if any of it is: BY_MASS the fraction `part` of its mass, else `count`
// tokens (at least 1 and at most what `from` holds). By radix descent over the
// keys. What is wanted of a mass is taken from the sum of its units, so that it is
// there to be found.
template <bool BY_MASS, typename R>
__device__ Cut radix_cut(const R& row, const Cut& from, uint32_t count, float part, Shared& s) {
  const float unit = wide_unit(row);
  uint32_t prefix = 0, mask = 0;  // the key's bits found so far, and which they are
  uint64_t left = count;
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (threadIdx.x < 256) s.wide_bins[threadIdx.x] = 0;
    __syncthreads();
    row.each([&](int i, float l) {
      const uint32_t k = key_of(l);
      if ((k & mask) == prefix && from.has(l, i)) atomicAdd(&s.wide_bins[(k >> shift) & 255], units<BY_MASS, uint64_t>(row, l, unit));
    });
    __syncthreads();
    // Thread t has bin 255 - t, of the largest keys first.
    const uint64_t mine = threadIdx.x < 256 ? s.wide_bins[255 - threadIdx.x] : 0;
    const uint64_t before = group_before(mine, s.list);
    if (BY_MASS && shift == 24) {
      if (threadIdx.x == kThreads - 1) s.entry = before + mine;  // the whole, at least the largest logit's
      __syncthreads();
      left = fraction(part, s.entry);
      __syncthreads();
    }
    if (before < left && before + mine >= left) {
      s.pick = 255 - threadIdx.x;
      s.entry = left - before;
    }
    __syncthreads();
    prefix |= s.pick << shift;
    mask |= 255u << shift;
    left = s.entry;
    __syncthreads();
  }
  // What is left of the tokens with exactly this key, by index: how many tokens
  // that is (they count the same), then where the last of them lies. A wave
  // looks at a run of the row.
  const float edge = value_of(prefix);
  const uint64_t each = max(units<BY_MASS, uint64_t>(row, edge, unit), uint64_t{1});
  const uint32_t want = static_cast<uint32_t>((left + each - 1) / each);
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int run = ((row.vocab + kWaves - 1) / kWaves + 63) / 64 * 64;
  const int t0 = w * run, t1 = min(t0 + run, row.vocab);
  auto hits = [&](int i) {
    const float l = i < t1 ? row.at(i) : 0.f;
    return __ballot(i < t1 && l == edge && from.has(l, i));
  };
  uint32_t mine = 0;
  for (int i = t0 + lane; i - lane < t1; i += 64) mine += __popcll(hits(i));
  if (lane == 0) s.u32[w] = mine;
  if (threadIdx.x == 0) s.pick = static_cast<uint32_t>(row.vocab - 1);
  __syncthreads();
  uint32_t seen = 0;
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
  const Cut cut{edge, s.pick};
  __syncthreads();
  return cut;
}

// The same by bins of equal width below M: as far as the row reaches (`low`),
// at most 24 T (where w is 4e-11); the last bin takes what lies beyond. False
// where that bin holds the cut, or the cut's bin too many logits. With U of 32
// bits, `want` of the units is looked for, else the fraction `part` of their sum.
template <bool BY_MASS, typename U, typename R>
__device__ __forceinline__ bool bins_cut(const R& row, float low, const Cut& from, U want, float part, float unit,
                                         Shared& s, Cut& cut) {
  U *bins, *slot;
  if constexpr (sizeof(U) == 4) {
    bins = s.bins;
    slot = s.u32;
  } else {
    bins = s.wide_bins;
    slot = s.list;
  }
  const float scale = (kBins - 1) / fmaxf(fminf(24.0f * row.temperature, row.top - low), 1e-30f);
  auto bin_of = [&](float l) {
    return static_cast<int>(__builtin_amdgcn_fmed3f((l - row.ref) * -scale, 0.f, kBins - 1.0f));
  };
  for (int i = threadIdx.x; i < kBins; i += kThreads) bins[i] = 0;
  __syncthreads();
  if (BY_MASS && from.edge == -__builtin_inff()) {  // everything; beyond the row's end the mass is 0
    row.each([&](int, float l) { atomicAdd(&bins[bin_of(l)], units<BY_MASS, U>(row, l, unit)); });
  } else {
    row.each([&](int i, float l) {
      if (from.has(l, i)) atomicAdd(&bins[bin_of(l)], units<BY_MASS, U>(row, l, unit));
    });
  }
  __syncthreads();
  const U b0 = bins[2 * threadIdx.x], b1 = bins[2 * threadIdx.x + 1];
  const U before = group_before(b0 + b1, slot);
  if constexpr (sizeof(U) == 8) {
    if (threadIdx.x == kThreads - 1) s.entry = before + b0 + b1;
    __syncthreads();
    want = fraction(part, s.entry);
  }
  if (threadIdx.x == 0) {
    s.pick = kBins - 1;  // rounding may leave the sum short of `want`
    s.n = 0;
  }
  __syncthreads();
  if (before < want && before + b0 + b1 >= want) {
    const bool second = before + b0 < want;
    s.pick = 2 * threadIdx.x + second;
    s.left = want - before - (second ? b0 : 0);
  }
  __syncthreads();
  const int bin = static_cast<int>(s.pick);
  const U left = static_cast<U>(s.left);
  if (bin < kBins - 1) {
    // Logits near the bin's range first (two comparisons), then the bin itself:
    // half a bin and four roundings of M wide of it, and bin 0 has no upper end.
    const float slack = 0.5f / scale + 4.8e-7f * fabsf(row.ref);
    const float high = bin == 0 ? __builtin_inff() : row.ref - bin / scale + slack;
    const float least = row.ref - (bin + 1) / scale - slack;
    row.each_pack([&](int i, const auto& q) {
      bool any = false;
#pragma unroll
      for (int e = 0; e < R::kE; ++e) any |= q.at(e) <= high && q.at(e) >= least;
      if (!any) return;
      for (uint32_t hits = q.which([&](float l) { return l <= high && l >= least; }); hits != 0; hits &= hits - 1) {
        const int e = __builtin_ctz(hits);
        const float l = q.pick(e);
        if (bin_of(l) == bin && from.has(l, i + e)) append(s, l, i + e);
      }
    });
    __syncthreads();
    const int n = static_cast<int>(s.n);
    __syncthreads();
    if (n <= kThreads) {
      const uint64_t e = sorted_entry(s, n);
      const bool in = static_cast<int>(threadIdx.x) < n;
      const U unit_here = in ? units<BY_MASS, U>(row, value_of(e >> 32), unit) : 0;
      const U at = group_before(unit_here, slot);
      if (in && at < left && at + unit_here >= left) s.entry = e;
      __syncthreads();
      cut = Cut{value_of(s.entry >> 32), 0xffffffffu - static_cast<uint32_t>(s.entry)};
      __syncthreads();
      return true;
    }
  }
  __syncthreads();
  return false;
}

// Masses in 32 bits where that is near enough: their units are 2^-31 of the
// whole, `total`, so the cut is off by half a unit a logit at most. 50280 bf16
// logits, 256 rows: 43 us, with 64 bits 46.
template <bool BY_MASS, typename R>
__device__ __forceinline__ Cut find_cut(const R& row, float low, const Cut& from, uint32_t count, float part,
                                        float total, Shared& s) {
  Cut cut;
  bool found;
  if (!BY_MASS || row.vocab * 0x1p-28f <= fminf(1.0f - part, 0x1p-9f)) {  // 16 vocab / 2 units
    const uint32_t want = BY_MASS ? static_cast<uint32_t>(fmaxf(ceilf(part * 0x1p31f), 1.0f)) : count;
    found = bins_cut<BY_MASS, uint32_t>(row, low, from, want, part, BY_MASS ? 0x1p31f / total : 1.0f, s, cut);
  } else {
    found = bins_cut<BY_MASS, uint64_t>(row, low, from, 0, part, wide_unit(row), s, cut);
  }
  return found ? cut : radix_cut<BY_MASS>(row, from, count, part, s);
}

// The largest key of the threads' maxima that at least `want` of them reach,
// or one a little lower: bisection by the first wave, the others wait.
__device__ __forceinline__ uint32_t maxima_key(Shared& s, int want) {
  if (threadIdx.x < 64) {
    uint32_t k[kThreads / 64];
#pragma unroll
    for (int j = 0; j < kThreads / 64; ++j) k[j] = key_of(s.tops[j * 64 + threadIdx.x]);
    uint32_t lo = 0xffffffffu, hi = 0;
#pragma unroll
    for (int j = 0; j < kThreads / 64; ++j) {
      lo = min(lo, k[j]);
      hi = max(hi, k[j]);
    }
    for (int o = 32; o > 0; o >>= 1) {
      lo = min(lo, static_cast<uint32_t>(__shfl_xor(lo, o)));
      hi = max(hi, static_cast<uint32_t>(__shfl_xor(hi, o)));
    }
    hi += 1;  // all reach lo; fewer than `want` reach hi
    while (hi - lo > 1) {
      const uint32_t mid = lo + (hi - lo) / 2;
      int n = 0;
#pragma unroll
      for (int j = 0; j < kThreads / 64; ++j) n += __popcll(__ballot(k[j] >= mid));
      if (n < want) {
        hi = mid;
      } else {
        lo = mid;
        if (n <= want + want / 16 + 4) break;
      }
    }
    if (threadIdx.x == 0) s.pick = lo;
  }
  __syncthreads();
  const uint32_t key = s.pick;
  __syncthreads();
  return key;
}

// ---- the race ----------------------------------------------------------------------------------

constexpr float kLeastNoise = 1.17549435e-38f;
__device__ __forceinline__ float noise_at(const float* noise, int i) { return fmaxf(noise[i], kLeastNoise); }

// E values of noise from i on; beyond the row's end 1.
template <int E>
__device__ __forceinline__ void load_noise(const float* noise, int i, int vocab, float (&q)[E]) {
  if (i + E <= vocab) {
#pragma unroll
    for (int e = 0; e < E; e += 4) {
      float q4[4];
      ld4_elem<float>(noise, i + e, q4);
#pragma unroll
      for (int x = 0; x < 4; ++x) q[e + x] = q4[x];
    }
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) q[e] = i + e < vocab ? noise[i + e] : 1.0f;
  }
}

// The workgroup's largest score and, of those who hold it, the lowest index.
template <int WAVES = kWaves>
__device__ __forceinline__ uint32_t winner(float score, uint32_t i, float* f32, uint32_t* u32) {
  const float top = group_max<WAVES>(score, f32);
  return group_min<WAVES>(score == top ? i : 0xffffffffu, u32);
}

// Scores are compared as log2(w / noise) first. Both logarithms are off by less
// than 150 x 2^-22, so whatever may be the winner lies within kNearLog, log2 of
// 1 / kNear, of the best.
constexpr float kNearLog = 1.7611e-4f;
template <typename R> __device__ __forceinline__ float fast_score(const R& row, float l, float noise) {
  return row.steps(l) - __builtin_amdgcn_logf(fmaxf(noise, kLeastNoise));
}

// A thread's best pack by its largest fast score, where, and the second best.
struct Best {
  float best = -__builtin_inff(), second = -__builtin_inff();
  int at = 0;
  __device__ __forceinline__ void see(float score, int i) {
    second = __builtin_amdgcn_fmed3f(best, second, score);  // second <= best
    at = score > best ? i : at;
    best = fmaxf(best, score);
  }
};

// The winner of the kept logits of a row.
// CUT: there are cuts; otherwise every logit is kept.
template <bool CUT, typename T>
__device__ __forceinline__ uint32_t race(const Row<T>& row, const Cut& kept, float min_p, const float* noise,
                                         Shared& s) {
  constexpr int kAhead = 2, E = kPer<T>;
  const float inf = __builtin_inff();
  const float above = value_of(key_of(kept.edge) + 1);  // the next logit above the edge; NaN above infinity
  const float least = __builtin_amdgcn_logf(min_p);
  // The fast scores of a pack, -inf for a logit that is not kept.
  auto scores = [&](int i, const Pack<T>& p, const float (&q)[E], float (&score)[E]) {
#pragma unroll
    for (int e = 0; e < E; ++e) score[e] = fast_score(row, p.at(e), q[e]);
    if constexpr (CUT) {
      const int last = static_cast<int>(kept.last);
      if (i <= last && last < i + E - 1) {
#pragma unroll
        for (int e = 0; e < E; ++e) score[e] = p.at(e) >= (i + e <= last ? kept.edge : above) ? score[e] : -inf;
      } else {
        const float edge = i <= last ? kept.edge : above;
#pragma unroll
        for (int e = 0; e < E; ++e) score[e] = p.at(e) >= edge ? score[e] : -inf;
      }
      if (min_p > 0.f) {
        // What lies too near min-p to tell is left to the weight itself.
        uint32_t hits = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float x = row.steps(p.at(e)) - least;
          score[e] = x >= -kNearLog ? score[e] : -inf;
          hits |= x >= -kNearLog && x <= kNearLog ? 1u << e : 0u;
        }
        for (; hits != 0; hits &= hits - 1) {
          const int at = __builtin_ctz(hits);
          if (row.weight(p.pick(at)) >= min_p) continue;
#pragma unroll
          for (int e = 0; e < E; ++e) score[e] = e == at ? -inf : score[e];
        }
      }
    }
  };
  auto load = [&](int i, Pack<T>& p, float (&q)[E]) {
    p = load_pack(row.logits, i, row.vocab);
    load_noise<E>(noise, i, row.vocab, q);
  };
  Best b;
  for (int i0 = threadIdx.x * E; i0 < row.vocab; i0 += kAhead * kThreads * E) {
    Pack<T> p[kAhead];
    float q[kAhead][E];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) load(i0 + j * kThreads * E, p[j], q[j]);
    if (row.odd) {
#pragma unroll
      for (int j = 0; j < kAhead; ++j) p[j] = clean(p[j]);
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      float score[E], most = -inf;
      scores(i0 + j * kThreads * E, p[j], q[j], score);
#pragma unroll
      for (int e = 0; e < E; ++e) most = __builtin_elementwise_maximum(most, score[e]);
      b.see(most, i0 + j * kThreads * E);
    }
  }
  const float bar = group_max(b.best, s.f32) - kNearLog;
  float score = -1.0f;
  uint32_t at = 0xffffffffu;
  if (b.best >= bar) {
    // The near ones of the best pack, or of all where another comes near it too.
    const bool all = b.second >= bar;
    for (int i = all ? static_cast<int>(threadIdx.x) * E : b.at; i < row.vocab; i += kThreads * E) {
      Pack<T> p;
      float q[E], fast[E];
      load(i, p, q);
      if (row.odd) p = clean(p);
      scores(i, p, q, fast);
      uint32_t hits = 0;
#pragma unroll
      for (int e = 0; e < E; ++e) hits |= fast[e] >= bar ? 1u << e : 0u;
      for (; hits != 0; hits &= hits - 1) {
        const int w = i + __builtin_ctz(hits);
        const float l = row.at(min(w, row.vocab - 1));
        if (w >= row.vocab || (CUT && (!kept.has(l, w) || !(row.weight(l) >= min_p)))) continue;
        const float exact = row.weight(l) / noise_at(noise, w);
        if (exact > score) {
          score = exact;
          at = static_cast<uint32_t>(w);
        }
      }
      if (!all) break;
    }
  }
  return winner(score, at, s.f32, s.u32);
}

template <typename T> __global__ __launch_bounds__(kThreads) void sample_row_kernel(const SampleParams p) {
  __shared__ Shared s;
  const int64_t r = p.first + blockIdx.x;
  Row<T> row;
  row.logits = static_cast<const T*>(p.logits) + r * p.sl;
  row.vocab = static_cast<int>(p.vocab);
  const float temperature = p.temperature_rows != nullptr ? p.temperature_rows[r] : p.temperature;
  int k = p.top_k_rows != nullptr ? p.top_k_rows[r] : p.top_k;
  const float top_p = p.top_p_rows != nullptr ? p.top_p_rows[r] : p.top_p;
  const float min_p = fminf(p.min_p_rows != nullptr ? p.min_p_rows[r] : p.min_p, 1.0f);
  if (k < 0 || k >= row.vocab) k = 0;  // off

  const float inf = __builtin_inff();
  float m = -inf, low = inf;
  // By v_maximum3_f32 and v_minimum3_f32, half an instruction a logit; a NaN
  // comes through, and the thread looks again.
  auto range = [&](bool clean_first) {
    m = -inf;
    low = inf;
    row.odd = clean_first;
    row.each_pack([&](int i, const Pack<T>& q) {
#pragma unroll
      for (int e = 0; e < kPer<T>; ++e) {
        m = __builtin_elementwise_maximum(m, q.at(e));
        low = __builtin_elementwise_minimum(low, i + kPer<T> <= row.vocab || i + e < row.vocab ? q.at(e) : inf);
      }
    });
  };
  range(false);
  const bool bad = m != m;
  if (bad) range(true);
  if ((threadIdx.x & 63) == 0) s.odd[threadIdx.x >> 6] = 0;
  if (bad) s.odd[threadIdx.x >> 6] = 1;
  s.tops[threadIdx.x] = m;
  m = group_max(m, s.f32);
  row.odd = __ballot(s.odd[threadIdx.x & (kWaves - 1)] != 0) != 0;
  if (m == -inf) {
    if (threadIdx.x == 0) {
      p.token[r] = -1;
      if (p.logprob != nullptr) p.logprob[r] = -inf;
    }
    return;
  }
  const bool greedy = !(temperature > 0.f);
  const bool few = !greedy && k > 0 && k <= kListK;
  const bool by_p = !greedy && top_p < 1.0f;
  const bool by_min = !greedy && !few && k == 0 && min_p > 0.f;
  const bool list = few || by_min || (by_p && k == 0);
  row.set(m, greedy ? 1.0f : temperature);
  // One more look at the row: the sums of exp(l - M), for the log-probability,
  // and of the weights, where top-p is asked without top-k; the lowest index of
  // M for T <= 0; the short list.
  const bool sum1 = p.logprob != nullptr, sum_t = by_p && k == 0;
  // The list's lowest logit: without top-k not below min-p's, with half a
  // percent of the weight and four roundings of M to spare.
  float from = inf;
  bool least = false;  // the list is min-p's
  if (list && row.vocab > kThreads) {
    if (few || by_p) from = value_of(maxima_key(s, few ? k : kTryK));
    const float by = by_min ? row.ref + row.temperature * (logf(min_p) - 0.005f) - 4.8e-7f * fabsf(row.ref) : -inf;
    least = by_min && (!by_p || by >= from);
    if (least) from = by;
  } else if (list) {
    from = -inf;
  }
  if (threadIdx.x == 0) s.n = 0;
  __syncthreads();
  float total1 = 0.f, total = 0.f;
  uint32_t token = 0xffffffffu;
  if (sum1 || list || greedy) {
    // What is looked for is rare: a pack's largest logit says whether it is there.
    const bool one = row.temperature == 1.0f, both = sum_t && !one;
    const float look = greedy ? m : from;
    row.each_pack([&](int i, const Pack<T>& q) {
      float high = -inf;
#pragma unroll
      for (int e = 0; e < kPer<T>; ++e) high = __builtin_elementwise_maximum(high, q.at(e));
      if (high >= look) {
        uint32_t hits = q.which([&](float l) { return l >= look; });
        if (i + kPer<T> > row.vocab) hits &= (1u << (row.vocab - i)) - 1;
        if (greedy) {
          if (hits != 0) token = min(token, static_cast<uint32_t>(i + __builtin_ctz(hits)));
          hits = 0;
        }
        for (; hits != 0; hits &= hits - 1) append(s, q.pick(__builtin_ctz(hits)), i + __builtin_ctz(hits));
      }
      if (sum1) {
#pragma unroll
        for (int e = 0; e < kPer<T>; ++e) total1 += upto1(fast_exp2((q.at(e) - row.ref) * kLog2e));
      }
      if (both) {
#pragma unroll
        for (int e = 0; e < kPer<T>; ++e) total += row.weight_fast(q.at(e));
      }
    });
    if (sum1) total1 = group_fsum(total1, s.f32);
    if (sum_t && one && !sum1) row.each([&](int, float l) { total += row.weight_fast(l); });
    if (sum_t) total = one && sum1 ? total1 : group_fsum(total, s.f32);
    __syncthreads();
  }
  if (greedy) {
    token = group_min(token, s.u32);
  } else {
    const float* noise = p.noise + r * p.sn;
    const float part = fmaxf(top_p, 0.f);
    const int n = static_cast<int>(s.n);
    __syncthreads();
    if (list && n <= kThreads) {
      const bool in = static_cast<int>(threadIdx.x) < n;
      bool holds = few || least || row.vocab <= kThreads;
      if (!holds) {
        // In integers: the list's order, not yet sorted, is another from call to call.
        const uint32_t mass = in ? units<true, uint32_t>(row, value_of(s.list[threadIdx.x] >> 32), 0x1p31f / total) : 0;
        holds = group_usum(mass, s.u32) > static_cast<uint32_t>(part * (2.0f - kNear) * 0x1p31f);
      }
      if (holds) {
        const uint64_t e = sorted_entry(s, n);
        const float w = in ? row.weight(value_of(e >> 32)) : 0.f;
        const uint32_t i = 0xffffffffu - static_cast<uint32_t>(e);
        bool keep = in && (!few || static_cast<int>(threadIdx.x) < k);
        if (by_p) {  // sums in the list's order, which is always the same
          const float mass = keep ? w : 0.f;
          const float all = few ? group_fsum(mass, s.f32) : total;
          keep = group_before(mass, s.f32) < part * all && keep;
        }
        keep = (keep && w >= min_p) || threadIdx.x == 0;
        token = winner(keep ? w / noise_at(noise, static_cast<int>(i)) : -1.0f, i, s.f32, s.u32);
      }
    }
    if (token == 0xffffffffu) {
      Cut kept{-inf, static_cast<uint32_t>(row.vocab - 1)};  // everything
      if (k > 0 || by_p) low = -group_max(-low, s.f32);
      if (k > 0) {
        kept = find_cut<false>(row, low, kept, static_cast<uint32_t>(k), 0.f, 0.f, s);
        if (by_p) {
          row.each([&](int i, float l) { total += kept.has(l, i) ? row.weight_fast(l) : 0.f; });
          total = group_fsum(total, s.f32);
        }
      }
      if (by_p) kept = find_cut<true>(row, low, kept, 0, part, total, s);
      token = k > 0 || by_p || min_p > 0.f ? race<true>(row, kept, min_p, noise, s)
                                           : race<false>(row, kept, min_p, noise, s);
      if (token == 0xffffffffu) {  // no score is a number (an infinite logit over infinite noise): the first token
        row.each([&](int i, float l) { token = l == m ? min(token, static_cast<uint32_t>(i)) : token; });
        token = group_min(token, s.u32);
      }
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

// ---- rows that nothing cuts, in slices -----------------------------------------------------------

constexpr int kSliceThreads = 512, kSliceMost = 64;  // threads, and slices of a row

// What a slice leaves for its row.
struct Slice {
  float top, sum;  // the largest logit; the sum of exp(l - top)
  uint32_t at;     // its winner, or for T <= 0 the lowest index of `top`
};

// The slice's packs of logits, and of noise, all on their way at once.
template <typename T, bool GREEDY>
__global__ __launch_bounds__(kSliceThreads) void sample_slice_kernel(const SampleParams p, int slices) {
  constexpr int E = kPer<T>, NP = kSampleSlice / (kSliceThreads * E);
  __shared__ float f32[kSliceThreads / 64];
  __shared__ uint32_t u32[kSliceThreads / 64];
  const uint32_t group = static_cast<uint32_t>(p.first) + blockIdx.x;
  const int64_t r = group / slices;
  const int first = static_cast<int>(group % slices) * kSampleSlice + static_cast<int>(threadIdx.x) * E;
  Row<T> row;
  row.logits = static_cast<const T*>(p.logits) + r * p.sl;
  row.vocab = static_cast<int>(p.vocab);
  const float* noise = p.noise + r * p.sn;
  Pack<T> l[NP];
  float q[GREEDY ? 1 : NP][E];
#pragma unroll
  for (int j = 0; j < NP; ++j) {
    const int i = first + j * kSliceThreads * E;
    l[j] = load_pack(row.logits, i, row.vocab);
    if constexpr (!GREEDY) load_noise<E>(noise, i, row.vocab, q[j]);
  }
  const float inf = __builtin_inff();
  float m = -inf;
  auto top = [&] {
    m = -inf;
#pragma unroll
    for (int j = 0; j < NP; ++j)
#pragma unroll
      for (int e = 0; e < E; ++e) m = __builtin_elementwise_maximum(m, l[j].at(e));
  };
  top();
  if (__ballot(m != m) != 0) {
#pragma unroll
    for (int j = 0; j < NP; ++j) l[j] = clean(l[j]);
    top();
  }
  m = group_max<kSliceThreads / 64>(m, f32);
  row.set(m, GREEDY ? 1.0f : p.temperature);
  float sum = 0.f, score = -1.0f;
  uint32_t at = 0xffffffffu;
  Best b;
#pragma unroll
  for (int j = 0; j < NP; ++j) {
    const int i = first + j * kSliceThreads * E;
    float most = -inf;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float v = l[j].at(e);
      sum += upto1(fast_exp2((v - row.ref) * kLog2e));
      if constexpr (GREEDY) at = v == m ? min(at, static_cast<uint32_t>(i + e)) : at;
      else most = __builtin_elementwise_maximum(most, fast_score(row, v, q[j][e]));
    }
    if constexpr (!GREEDY) b.see(most, i);
  }
  sum = group_fsum<kSliceThreads / 64>(sum, f32);
  if constexpr (GREEDY) {
    at = group_min<kSliceThreads / 64>(at, u32);
  } else {
    const float bar = group_max<kSliceThreads / 64>(b.best, f32) - kNearLog;
    // The best pack's logits, or all the thread's where another comes near it.
    if (b.best >= bar) {
      const bool all = b.second >= bar;
      const int most = all ? NP * E : E;
#pragma unroll 1
      for (int n = 0; n < most; ++n) {
        const int i = (all ? first + n / E * kSliceThreads * E : b.at) + n % E;
        if (i >= row.vocab) continue;
        const float exact = row.weight(row.at(i)) / noise_at(noise, i);
        if (exact > score) {
          score = exact;
          at = static_cast<uint32_t>(i);
        }
      }
    }
    at = winner<kSliceThreads / 64>(score, at, f32, u32);
  }
  if (threadIdx.x == 0) static_cast<Slice*>(p.slices)[group] = Slice{m, m == -inf ? 0.f : sum, at};
}

// A row's token from its slices' winners, one lane each.
template <typename T, bool GREEDY>
__global__ __launch_bounds__(64) void sample_join_kernel(const SampleParams p, int slices) {
  const int64_t r = p.first + blockIdx.x;
  const int lane = threadIdx.x;
  const float inf = __builtin_inff();
  const Slice mine = lane < slices ? static_cast<const Slice*>(p.slices)[r * slices + lane] : Slice{-inf, 0.f, 0u};
  float m = mine.top;
  for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
  if (m == -inf) {
    if (lane == 0) {
      p.token[r] = -1;
      if (p.logprob != nullptr) p.logprob[r] = -inf;
    }
    return;
  }
  Row<T> row;
  row.logits = static_cast<const T*>(p.logits) + r * p.sl;
  row.vocab = static_cast<int>(p.vocab);
  row.set(m, GREEDY ? 1.0f : p.temperature);
  // Slices without a logit above -inf, or with none near M, lose or have no winner.
  const bool in = lane < slices && mine.top > -inf && mine.at < static_cast<uint32_t>(row.vocab);
  float score = -1.0f, sum = 0.f;
  if (in) {
    if constexpr (GREEDY) score = mine.top == m ? 1.0f : 0.f;
    else score = row.weight(row.at(static_cast<int>(mine.at))) / noise_at(p.noise + r * p.sn, static_cast<int>(mine.at));
    sum = mine.sum * (mine.top == m ? 1.0f : exp_acc(mine.top - m));
  }
  float best = score;
  for (int o = 32; o > 0; o >>= 1) best = fmaxf(best, __shfl_xor(best, o));
  uint32_t token = in && score == best ? mine.at : 0xffffffffu;
  for (int o = 32; o > 0; o >>= 1) token = min(token, static_cast<uint32_t>(__shfl_xor(token, o)));
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
  if (lane == 0) {
    p.token[r] = static_cast<int64_t>(token);
    if (p.logprob != nullptr && token < static_cast<uint32_t>(row.vocab)) {
      const float l = row.at(static_cast<int>(token));
      p.logprob[r] = (l == m ? 0.f : l - m) - logf(sum);
    }
  }
}

template <typename T, bool GREEDY> void launch_slices(SampleParams p, int64_t slices, hipStream_t st) {
  const int n = static_cast<int>(slices);
  launch_all(p.rows * slices, kSliceThreads, [&](int64_t first, unsigned groups) {
    p.first = first;
    hipLaunchKernelGGL((sample_slice_kernel<T, GREEDY>), dim3(groups), dim3(kSliceThreads), 0, st, p, n);
  });
  launch_all(p.rows, 64, [&](int64_t first, unsigned groups) {
    p.first = first;
    hipLaunchKernelGGL((sample_join_kernel<T, GREEDY>), dim3(groups), dim3(64), 0, st, p, n);
  });
}

template <typename T> void launch(SampleParams p, hipStream_t st) {
  const int64_t slices = sample_slices(p);
  if (slices > 0) return p.temperature > 0.f ? launch_slices<T, false>(p, slices, st) : launch_slices<T, true>(p, slices, st);
  launch_all(p.rows, kThreads, [&](int64_t first, unsigned groups) {
    p.first = first;
    hipLaunchKernelGGL(sample_row_kernel<T>, dim3(groups), dim3(kThreads), 0, st, p);
  });
}

}  // namespace

// Slices of a row (0: none, the row kernel): where one setting holds for all
// rows and cuts nothing, and a row has at most a lane's worth of slices. A row
// of one slice needs no second launch: 8 x 1000 take 9 us with one, 12 with two.
int64_t sample_slices(const SampleParams& p) {
  const bool rows_alike = p.temperature_rows == nullptr && p.top_k_rows == nullptr && p.top_p_rows == nullptr &&
                          p.min_p_rows == nullptr;
  const bool greedy = p.temperature <= 0.f;
  const bool uncut = greedy || ((p.top_k == 0 || p.top_k >= p.vocab) && p.top_p >= 1.0f && p.min_p <= 0.f);
  const int64_t n = (p.vocab + kSampleSlice - 1) / kSampleSlice;
  return rows_alike && uncut && n > 1 && n <= kSliceMost && p.rows * n <= INT32_MAX ? n : 0;
}
size_t sample_workspace(const SampleParams& p) { return sizeof(Slice) * p.rows * sample_slices(p); }

hipError_t sample_launch(SampleParams p, hipStream_t st) {
  if (p.dtype == MCPU_F32) launch<float>(p, st);
  else if (p.dtype == MCPU_BF16) launch<bf16>(p, st);
  else launch<f16>(p, st);
  return hipGetLastError();
}

}  // namespace mcpu
