// Losses of a language model's head on gfx950, without its logits kept. With
// s_tv = h_t . w_v over tokens t and vocabulary v, c = 1 / temperature:
//   L_t = log sum_v exp(c s_tv)
//   cross entropy  loss_t = L_t - s_{t, y_t}                                  (c = 1)
//   distillation   q_t = softmax(c teacher_t) over the ids in the vocabulary,
//                  loss_t = (sum_k q_k log q_k + L_t - sum_k q_k c s_{t, id_k}) / c^2
// and, with g_t the gradient of loss_t and e_t that of L_t,
//   ds_tv = a_t exp(c s_tv - L_t) - b_t sum_{k: id_k = v} q_tk
//   a = g + e, b = g (cross entropy, q = 1);  a = b = g / c (distillation)
//   dhidden = ds weight,  dweight = ds^T hidden.
//
// Forward: one product of the rows that count, whose epilogue keeps a maximum and a
// sum of 128 vocabulary rows per token, then one pass that joins these. A target's
// logit is taken from the product, and out of its sums: a loss near 0 then has its
// digits. The products of hidden with a teacher's ids are formed by themselves.
// Backward: a piece of the vocabulary at a time, the product again, now with ds in
// 16 bits as its result (float32: two f16 pieces), the ids' places put right, and
// the two products of the gradients over it. dweight's reads hidden's rows times their
// ds's unit over the largest, rounded once more to the kept type (loss_coef_kernel has
// why, kLeastUnit how far). Rows that do not count take part in no product, so nothing in
// them, NaN included, reaches another row.
//
// Three ways to the logits, by how many tiles there are:
//   tiles of 256 x 256     bound by the matrix cores at the clock that power leaves
//                          them: 16384 x 50280 x 768 bf16 1.13-1.25 ms, 1010-1120 TFLOP/s
//   blocks of 64 x 128     up to 512 of them, where tiles would not fill the GPU
//   up to 64 tokens        the same kernel on the rows as they come and one more that does the
//                          rest: bound by reading weight, 4.4 TB/s
// loss_plan has the rule and both sides. The gradients' products are tiles always.
//
// Everything is summed in float32, in an order that depends on the sizes and on the
// number of rows that count alone: no atomics add.
#include "launch.h"
#include "lm_math.h"
#include "tile_product.h"

namespace mcpu {
namespace {

// ds is kept as ds / unit times this: f16's steps are then 2^-37 of the unit.
template <typename E> constexpr float kUp = std::is_same_v<E, bf16> ? 1.f : 8192.f;
// f16 pieces: the least unit of a row beside the largest. dweight's product takes unit / the largest from hidden's
// rows, whose largest magnitude is 2^13 or more: with 2^-16 of it left, their elements down to 2^-11 of the largest
// keep all bits of an f16. What is below goes to ds, whose largest of a row falls from 2^13 on. All of it to hidden,
// unscaled, left 4 bits of an element near 1 at a unit of 2^-20 and nothing at 2^-26; all of it to ds would do that
// to dhidden.
constexpr float kLeastUnit = 0x1p-16f;

__device__ __forceinline__ int64_t id_at(const LossParams& p, int64_t i) {
  return p.ids64 ? static_cast<const int64_t*>(p.ids)[i] : static_cast<const int32_t*>(p.ids)[i];
}

// Microseconds of a product of `tiles` results of 256 KiB over `depths` each in
// `splits`: 256 workgroups at a time, at 4.7 TFLOP/s each with 6 us around a tile,
// and 4 TB/s for float32 results, written and read, where there are any.
template <typename I> __host__ __device__ inline float product_us(I tiles, I depths, I splits, bool apart) {
  const float rounds = static_cast<float>((tiles * splits + 255) / 256);
  return rounds * (static_cast<float>((depths + splits - 1) / splits) * 1.8f + 6.f) +
         (apart || splits > 1 ? static_cast<float>(tiles * splits) * 0.131f : 0.f);
}
// Splits that fill one to eight rounds of 256, or none, whichever takes least.
__host__ __device__ inline int splits_for(int64_t tiles, int64_t depths, bool apart) {
  if (tiles < 1 || tiles > kLossSplitTiles / 2) return 1;
  // In 32 bits, which the sizes left fit: the GPU divides 64 by a routine.
  const int t = static_cast<int>(tiles), d = static_cast<int>(depths);
  int best = 1;
  float least = product_us(t, d, 1, apart);
  const int most = d / 4 < kLossMostSplits ? d / 4 : kLossMostSplits;
  for (int rounds = 1; rounds <= 8; ++rounds) {
    const int s = 256 * rounds / t < most ? 256 * rounds / t : most;
    if (s < 2 || t * s > kLossSplitTiles) continue;
    const float us = product_us(t, d, s, apart);
    if (us < 0.97f * least) best = s, least = us;
  }
  return best;
}

// The power of two that brings a largest magnitude (as bits) to [2^13, 2^14), and its inverse.
__device__ __forceinline__ int up_exponent(uint32_t most) {
  if (most == 0) return 0;
  const int e = 13 - (static_cast<int>(most >> 23) - 127);
  return e > 120 ? 120 : e;
}
// exp(c (x - m)) is 2^(c x - m2), one multiply-add, with m2 = c m as rounded and its rounding (2^-9 at most) taken out
// of the sum. From here on that rounding is no small correction: such rows take the difference first.
constexpr float kFar = 0x1p16f;
__device__ __forceinline__ bool is_far(float m2) { return __builtin_fabsf(m2) >= kFar; }

// The largest power of two that is not above x.
__device__ __forceinline__ float power_below(float x) {
  return __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, x) & 0x7f800000u);
}
// The unit of a row that counts. One below the least becomes that by a power of two: its target's ds stays exact.
template <typename E> __device__ __forceinline__ float unit_of(const LossParams& p, int64_t i) {
  const float u = p.coef[3 * p.tpad + i], most = p.scal->unit;
  if (!(u > 0.f)) return most;
  if (std::is_same_v<E, bf16> || u >= most * kLeastUnit) return u;
  return __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, u) & 0x7fffffu) |
                                       __builtin_bit_cast(uint32_t, power_below(most * kLeastUnit)));
}
__device__ __forceinline__ float pow2(int e) { return __builtin_bit_cast(float, static_cast<uint32_t>(e + 127) << 23); }

// hi + lo of a scaled value; one that is not finite has no lo.
__device__ __forceinline__ void split_f16(float x, f16& hi, f16& lo) {
  hi = static_cast<f16>(x);
  const float rest = x - static_cast<float>(hi);
  lo = __builtin_fabsf(rest) < 65504.f ? static_cast<f16>(rest) : static_cast<f16>(0.f);
}

// ---- the teacher's distribution and products, which rows count ------------------------------

// h_t . w_v over a group of 16 lanes.
template <typename T> __device__ __forceinline__ float dot16(const T* h, const T* w, int64_t dim, int j) {
  float s = 0.f;
  int64_t i = j * 4;
  for (; i + 64 * 3 + 4 <= dim; i += 64 * 4) {
    float x[4][4], y[4][4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      ld4_elem<T>(h, i + u * 64, x[u]);
      ld4_elem<T>(w, i + u * 64, y[u]);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) s = fmaf(x[u][e], y[u][e], s);
  }
  for (; i < dim; i += 64) {
    float x[4], y[4];
    ld_upto4<T>(h, i, upto4(dim - i), x);
    ld_upto4<T>(w, i, upto4(dim - i), y);
#pragma unroll
    for (int e = 0; e < 4; ++e) s = fmaf(x[e], y[e], s);
  }
  return row_allreduce16(s);
}

// Distillation: a workgroup a token, 16 lanes a product.
template <typename T, int THREADS> __device__ __forceinline__ void teacher_row(const LossParams& p, int64_t t) {
  __shared__ float parts[THREADS / 64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int k = static_cast<int>(p.k);
  const float* teacher = p.teacher + t * k;
  const float c = 1.f / p.temperature;
  // An entry of -inf has no share; NaN has, and makes the row NaN.
  auto has = [&](int i) {
    const int64_t id = id_at(p, t * k + i);
    return id >= 0 && id < p.vocab && !(teacher[i] == -INFINITY);
  };
  // Every wave by itself.
  float m = -INFINITY;
  bool any = false;
  for (int i = lane; i < k; i += 64)
    if (has(i)) {
      any = true;
      m = fmaxf(m, teacher[i]);
    }
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) m = fmaxf(m, __shfl_xor(m, s));
  const bool keep = __any(any);
  float sum = 0.f;
  for (int i = lane; i < k; i += 64)
    if (has(i)) sum += exp_acc((teacher[i] - m) * c);
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) sum += __shfl_xor(sum, s);
  const float logsum = logf(sum), inv = 1.f / sum;
  // The products, and sum q (log q - c s).
  const int j = lane & 15;
  float cross = 0.f;
  for (int i = threadIdx.x >> 4; i < k; i += THREADS / 16) {
    float s = 0.f, q = 0.f;
    if (has(i)) {
      s = dot16<T>(static_cast<const T*>(p.hidden) + t * p.sh,
                   static_cast<const T*>(p.weight) + id_at(p, t * k + i) * p.sw, p.dim, j);
      const float x = (teacher[i] - m) * c;
      q = exp_acc(x) * inv;
      if (!(q == 0.f)) cross = fmaf(q, (x - logsum) - c * s, cross);
    }
    if (j == 0) {
      p.picked[t * k + i] = s;
      p.share[t * k + i] = q;
    }
  }
  cross += __shfl_xor(cross, 16);
  cross += __shfl_xor(cross, 32);
  if (lane == 0) parts[w] = cross;
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int i = 1; i < THREADS / 64; ++i) cross += parts[i];
  p.keep[t] = keep;
  p.cross[t] = cross;
}
template <typename T> __global__ __launch_bounds__(256) void loss_teacher_kernel(const LossParams p) {
  teacher_row<T, 256>(p, p.first + blockIdx.x);
}

__device__ __forceinline__ bool counts(const LossParams& p, int64_t t) {
  if (p.teacher != nullptr) return p.keep[t];
  const int64_t id = id_at(p, t);
  return id >= 0 && id < p.vocab && id != p.ignore;
}

// The rows that count, in order, then the others; one workgroup, 16 runs of 1024 rows at a time.
__global__ __launch_bounds__(1024) void loss_rows_kernel(const LossParams p) {
  __shared__ int32_t before[16][17];  // of a run's waves, then of all before them
  __shared__ int32_t runs[17];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int64_t kept = 0;
  for (int64_t t0 = 0; t0 < p.tokens; t0 += 16384) {
    uint32_t flags = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int64_t t = t0 + i * 1024 + threadIdx.x;
      if (t < p.tokens) flags |= static_cast<uint32_t>(counts(p, t)) << i;
    }
    unsigned long long mask[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      mask[i] = __ballot(flags >> i & 1);
      if (lane == 0) before[i][w] = __popcll(mask[i]);
    }
    __syncthreads();
    if (threadIdx.x < 16) {  // a run each
      int32_t sum = 0;
      for (int q = 0; q < 16; ++q) {
        const int32_t n = before[threadIdx.x][q];
        before[threadIdx.x][q] = sum;
        sum += n;
      }
      runs[threadIdx.x] = sum;
    }
    __syncthreads();
    int64_t at = kept;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int64_t t = t0 + i * 1024 + threadIdx.x;
      const int64_t mine = at + before[i][w] + __popcll(mask[i] & ((1ull << lane) - 1));  // that count before t
      if (t < p.tokens) p.rows[flags >> i & 1 ? mine : p.tokens - 1 - (t - mine)] = static_cast<int32_t>(t);
      at += runs[i];
    }
    kept = at;
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    p.rows[p.tokens] = static_cast<int32_t>(kept);
    p.scal->kept = static_cast<int32_t>(kept);
    p.scal->hmax = p.scal->wmax = 0;
  }
}

// ---- operands ----------------------------------------------------------------------------

// The largest finite magnitude of rows: two rows a wave at a time, 1024 elements of each on their way. 256
// workgroups of 16 waves, for one atomic each: one a wave, 8192 to one address, took 80 us. 8.5 us for hidden of
// 1021 x 1001 in f16.
template <typename T> __global__ __launch_bounds__(1024) void loss_most_kernel(const LossParams p, bool of_weight) {
  const int64_t rows = of_weight ? p.vocab : p.scal->kept;
  const int lane = threadIdx.x & 63;
  const int64_t waves = gridDim.x * 16ll;
  uint32_t most = 0;
  for (int64_t r = blockIdx.x * 16 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); r < rows; r += 2 * waves) {
    const T* row[2];
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const int64_t at = r + w * waves < rows ? r + w * waves : r;
      row[w] = of_weight ? static_cast<const T*>(p.weight) + at * p.sw
                         : static_cast<const T*>(p.hidden) + p.rows[at] * p.sh;
    }
    for (int64_t i0 = lane * 4; i0 < p.dim; i0 += 1024) {
      float v[2][4][4] = {};
#pragma unroll
      for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (i0 + u * 256 < p.dim) ld_upto4<T>(row[w], i0 + u * 256, upto4(p.dim - i0 - u * 256), v[w][u]);
#pragma unroll
      for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t b = __builtin_bit_cast(uint32_t, v[w][u][e]) & 0x7fffffffu;
            most = b < 0x7f800000u && b > most ? b : most;
          }
    }
  }
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) {
    const uint32_t o = __shfl_xor(most, s);
    most = o > most ? o : most;
  }
  __shared__ uint32_t tops[16];
  if (lane == 0) tops[threadIdx.x >> 6] = most;
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int i = 1; i < 16; ++i) most = tops[i] > most ? tops[i] : most;
  if (most > 0) atomicMax(of_weight ? &p.scal->wmax : &p.scal->hmax, most);
}

template <typename T> using Kept = std::conditional_t<std::is_same_v<T, float>, f16, T>;

// What hidden's rows of dweight's product are scaled by: its largest magnitude to [2^13, 2^14). bf16 has float32's range.
template <typename T> __device__ __forceinline__ int dweight_exponent(const LossParams& p) {
  if (std::is_same_v<T, float> || (std::is_same_v<T, f16> && p.hscaled != nullptr)) return up_exponent(p.scal->hmax);
  return 0;
}
template <typename T> __device__ __forceinline__ float dweight_up(const LossParams& p) {
  return pow2(dweight_exponent<T>(p));
}

// A row in the products' layout, zero behind its end: a wave a row, 64 elements at a time.
template <typename T>
__device__ __forceinline__ void lay_row(const T* from, void* to, int64_t at, int64_t piece, int64_t dim, int64_t dpad,
                                        float up, int lane) {
  for (int64_t i = lane * 4; i < dpad; i += 256) {
    float v[4] = {};
    if (from != nullptr && i < dim) ld_upto4<T>(from, i, upto4(dim - i), v);
    if constexpr (std::is_same_v<T, float>) {
      f16 hi[4], lo[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) split_f16(v[e] * up, hi[e], lo[e]);
      f16* out = static_cast<f16*>(to) + at + i;
#pragma unroll
      for (int e = 0; e < 4; ++e) out[e] = hi[e], out[piece + e] = lo[e];
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] *= up;
      st4_elem<T>(static_cast<T*>(to) + at, i, v);
    }
  }
}

template <typename T> __global__ __launch_bounds__(256) void loss_gather_kernel(const LossParams p) {
  const int64_t i = (p.first + blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t kept = p.scal->kept;
  if (i >= (kept + kLossTile - 1) / kLossTile * kLossTile) return;
  const float up = std::is_same_v<T, float> ? pow2(up_exponent(p.scal->hmax)) : 1.f;
  const int64_t t = i < kept ? p.rows[i] : 0;
  const T* from = i < kept ? static_cast<const T*>(p.hidden) + t * p.sh : nullptr;
  if (p.target != nullptr && (threadIdx.x & 63) == 0)
    p.target[i] = i < kept ? static_cast<int32_t>(id_at(p, t)) : -1;
  lay_row<T>(from, p.hrows, i * p.dpad, p.tpad * p.dpad, p.dim, p.dpad, up, threadIdx.x & 63);
  // The backward's, in the largest unit.
  if (p.hscaled != nullptr)
    lay_row<T>(from, p.hscaled, i * p.dpad, p.tpad * p.dpad, p.dim, p.dpad,
               dweight_up<T>(p) * (i < kept ? unit_of<Kept<T>>(p, i) / p.scal->unit : 0.f), threadIdx.x & 63);
}

template <typename T> __global__ __launch_bounds__(256) void loss_weight_kernel(const LossParams p) {
  const int64_t v = (p.first + blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (v >= p.vocab) return;
  if (p.laid != nullptr && v == 0 && (threadIdx.x & 63) == 0) *p.laid = p.scal->wmax;
  const float up = std::is_same_v<T, float> ? pow2(up_exponent(p.scal->wmax)) : 1.f;
  lay_row<T>(static_cast<const T*>(p.weight) + v * p.sw, p.wrows, v * p.dpad, p.vocab * p.dpad, p.dim, p.dpad, up,
             threadIdx.x & 63);
}

// ---- the products ---------------------------------------------------------------------------

template <typename T> constexpr int kRuns = std::is_same_v<T, float> ? 3 : 1;

// What takes the scaling of float32 operands back, and log2(e) c with it.
template <typename T> __device__ __forceinline__ float logit_back(const LossParams& p) {
  if constexpr (!std::is_same_v<T, float>) return 1.f;
  return pow2(-up_exponent(p.scal->hmax)) * pow2(-up_exponent(p.scal->wmax));
}
template <typename T> __device__ __forceinline__ float logit_scale(const LossParams& p) {
  return kLog2e / p.temperature * logit_back<T>(p);
}

__device__ __forceinline__ Operand rows_operand(const LossParams& p, const void* rows) {
  return {rows, p.dpad, p.tpad * p.dpad, p.tpad * p.dpad};
}
__device__ __forceinline__ Operand weight_operand(const LossParams& p, int64_t v0) {
  // In place, the rows end with dim = dpad elements.
  const int64_t ld = p.wrows != nullptr ? p.dpad : p.sw;
  const char* base = static_cast<const char*>(p.wrows != nullptr ? p.wrows : p.weight) + 2 * v0 * ld;
  return {base, ld, p.vocab * p.dpad, (p.vocab - v0 - 1) * ld + p.dpad};
}
__device__ __forceinline__ Operand grad_operand(const LossParams& p) {
  return {p.grad, p.vpiece, p.tpad * p.vpiece, p.tpad * p.vpiece};
}

// f takes each of a wave's accumulators of 32 tokens with its vocabulary row, less
// what the lane adds to it (4 for the upper half of the wave).
template <typename F> __device__ __forceinline__ void each_row(f32x16 (&x)[4], F&& f) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) x[i][e] = f(x[i][e], 32 * i + 8 * (e >> 2) + (e & 3));
}

// A lane's row among the wave's 128 from v0 on, as each_row counts, that is its token's target; -1 for none.
__device__ __forceinline__ int target_row(int32_t target, int64_t v0, int lane) {
  const int64_t at = target - v0;
  return at >= 0 && at < 128 && ((at >> 2) & 1) == lane >> 5 ? static_cast<int>(at) - 4 * (lane >> 5) : -1;
}

// Rows of the wave's 128 from v0 on that the vocabulary has, as each_row counts.
__device__ __forceinline__ int rows_left(const LossParams& p, int64_t v0, int lane) {
  const int64_t left = p.vocab - v0;
  return static_cast<int>(left < 0 ? 0 : left > 128 ? 128 : left) - 4 * (lane >> 5);
}

// Logits of a tile of 256 vocabulary rows (m) and 256 tokens (n): per token the
// maximum of each 128 rows and the sum relative to it; a target is left out and kept
// by itself, so that a loss near 0 has its digits.
template <typename T> __global__ __launch_bounds__(512, 2) void loss_logits_kernel(const LossParams p) {
  const int64_t kept = p.scal->kept;
  int64_t mt, nt;
  const int64_t mts = (p.vocab + kLossTile - 1) / kLossTile, nts = (kept + kLossTile - 1) / kLossTile;
  if (!tile_of(p.first + blockIdx.x, mts, nts, mt, nt)) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t v0 = mt * kLossTile + (wave >> 2) * kLossPart, t0 = nt * kLossTile + (wave & 3) * 64 + (lane & 31);
  // What the epilogue needs is on its way before the product.
  const float c = logit_scale<T>(p), back = logit_back<T>(p);
  const int32_t target[2] = {p.target != nullptr ? p.target[t0] : -1, p.target != nullptr ? p.target[t0 + 32] : -1};
  constexpr int runs = kRuns<T>;
  const ProductParams q = {weight_operand(p, 0), rows_operand(p, p.hrows), p.dpad, runs};
  MCPU_TILE_LDS(a0, b0, a1, b1);
  Acc acc;
  tile_product<Kept<T>, false, false>(q, mt * kLossTile, nt * kLossTile, 0,
                                      static_cast<int>(p.dpad / kLossDepth) * runs, a0, b0, a1, b1, acc);
  const int left = rows_left(p, v0, lane);
  if (mt * kLossTile + kLossTile > p.vocab) {
#pragma unroll
    for (int j = 0; j < 2; ++j) each_row(acc.v[j], [&](float x, int row) { return row < left ? x : -INFINITY; });
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int64_t t = t0 + j * 32;
    // Rare: one in V / 128 waves for each 32 tokens.
    const int at = target_row(target[j], v0, lane);
    if (__any(at >= 0)) {
      float own = 0.f;
      each_row(acc.v[j], [&](float x, int row) {
        own = row == at ? x : own;
        return row == at ? -INFINITY : x;
      });
      if (at >= 0) p.picked[t] = own * back;
    }
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) m = fmaxf(m, acc.v[j][i][e]);
    m = fmaxf(m, __shfl_xor(m, 32));
    // Relative to m * c as rounded, one multiply-add an element; then its rounding is taken out.
    const float m2 = m == -INFINITY ? 0.f : m * c;
    float s = 0.f;
    if (__any(is_far(m2))) {
      const float sub = m == -INFINITY ? 0.f : m;
      each_row(acc.v[j], [&](float x, int) {
        s += fast_exp2((x - sub) * c);
        return x;
      });
      s += __shfl_xor(s, 32);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) s += fast_exp2(fmaf(acc.v[j][i][e], c, -m2));
      s += __shfl_xor(s, 32);
      s = fmaf(s, -kLn2 * (m == -INFINITY ? 0.f : fmaf(m, c, -m2)), s);
    }
    if (lane < 32 && v0 < p.vocab) p.part[(v0 / kLossPart) * p.tpad + t] = make_float2(m * back, s);
  }
}

// The same product over a piece of the vocabulary, to ds in 16 bits.
template <typename T> __global__ __launch_bounds__(512, 2) void loss_grad_kernel(const LossParams p, int64_t vp) {
  using E = Kept<T>;
  const int64_t kept = p.scal->kept;
  int64_t mt, nt;
  if (!tile_of(p.first + blockIdx.x, p.vrows / kLossTile, (kept + kLossTile - 1) / kLossTile, mt, nt)) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t v0 = mt * kLossTile + (wave >> 2) * 128, t0 = nt * kLossTile + (wave & 3) * 64 + (lane & 31);
  const float c = logit_scale<T>(p);
  float a[2], b[2], m2[2];
  int32_t target[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int64_t t = t0 + j * 32;
    const float up = kUp<E> / unit_of<E>(p, t);
    a[j] = p.coef[t] * up;
    b[j] = p.coef[p.tpad + t] * up;
    m2[j] = p.coef[2 * p.tpad + t];
    target[j] = p.target != nullptr ? p.target[t] : -1;
  }
  constexpr int runs = kRuns<T>;
  const ProductParams q = {weight_operand(p, vp), rows_operand(p, p.hrows), p.dpad, runs};
  MCPU_TILE_LDS(a0, b0, a1, b1);
  Acc acc;
  tile_product<E, false, false>(q, mt * kLossTile, nt * kLossTile, 0, static_cast<int>(p.dpad / kLossDepth) * runs,
                                a0, b0, a1, b1, acc);
  const bool edge = vp + (mt + 1) * kLossTile > p.vocab || (nt + 1) * kLossTile > kept;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int64_t t = t0 + j * 32;
    if (__any(is_far(m2[j]))) {
      const float back = logit_back<T>(p), c0 = kLog2e / p.temperature, top = t < kept ? p.stat[t] : 0.f;
      each_row(acc.v[j], [&](float x, int) {
        return a[j] * fast_exp2(is_far(m2[j]) ? (x * back - top) * c0 : fmaf(x, c, -m2[j]));
      });
    } else {
      each_row(acc.v[j], [&](float x, int) { return a[j] * fast_exp2(fmaf(x, c, -m2[j])); });
    }
    const int at = target_row(target[j], vp + v0, lane);
    if (__any(at >= 0)) each_row(acc.v[j], [&](float x, int row) { return row == at ? b[j] : x; });
    if (edge) {
      const int left = t < kept ? rows_left(p, vp + v0, lane) : 0;
      each_row(acc.v[j], [&](float x, int row) { return row < left ? x : 0.f; });
    }
    uint16_t* out = static_cast<uint16_t*>(p.grad) + t * p.vpiece + v0 + 8 * (lane >> 5);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int g = 0; g < 4; g += 2) {
        // Four rows a lane become eight: the halves of the wave trade the second of two groups of eight.
        auto put = [&](const float* x, uint16_t* to) {
          uint32_t x0, x1, y0, y1;
          narrow4<E>(x, x0, x1);
          narrow4<E>(x + 4, y0, y1);
          const auto s0 = __builtin_amdgcn_permlane32_swap(x0, y0, false, false);
          const auto s1 = __builtin_amdgcn_permlane32_swap(x1, y1, false, false);
          const uint32_t r0 = s0[0], r1 = s1[0], r2 = s0[1], r3 = s1[1];
          *reinterpret_cast<u32x4*>(to + 32 * i + 8 * g) = u32x4{r0, r1, r2, r3};
        };
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = acc.v[j][i][4 * g + e];
        put(x, out);
        if constexpr (std::is_same_v<T, float>) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            f16 hi, lo;
            split_f16(x[e], hi, lo);
            x[e] = static_cast<float>(lo);
          }
          put(x, out + p.tpad * p.vpiece);
        }
      }
  }
}

// An entry's id, or -1 where it lies outside the vocabulary or there is none.
__device__ __forceinline__ int32_t in_vocab(const LossParams& p, int64_t i, bool any) {
  const int64_t id = any ? id_at(p, i) : -1;
  return id >= 0 && id < p.vocab ? static_cast<int32_t>(id) : -1;
}

// Distillation: the ids' places of ds, a_t exp(c s - L) less all shares of that id. A
// wave a row. In 16 bits that is formed anew, to be rounded once, but in far rows, where the
// two products' roundings would part `picked` from the row's sum. float32 takes p
// from the two pieces that are there: where p and its share are both near 1, their
// difference is as good as p agrees with the row's sum, and that is of the same
// product, while `picked` is a sum of its own.
template <typename T> __global__ __launch_bounds__(256) void loss_place_kernel(const LossParams p, int64_t vp) {
  using E = Kept<T>;
  const int lane = threadIdx.x & 63;
  const int64_t i = (p.first + blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (i >= p.scal->kept) return;
  const int64_t t = p.rows[i];
  const int k = static_cast<int>(p.k);
  const float up = kUp<E> / unit_of<E>(p, i), c = kLog2e / p.temperature;
  const float a = p.coef[i] * up, b = p.coef[p.tpad + i] * up, m2 = p.coef[2 * p.tpad + i];
  for (int e0 = 0; e0 < k; e0 += 64) {
    const int e = e0 + lane;
    const int32_t id = in_vocab(p, t * k + e, e < k);
    const int64_t v = id - vp;
    const bool here = id >= 0 && v >= 0 && v < p.vrows;
    if (!__any(here)) continue;
    // All entries of that id, 64 at a time from the lanes that hold them.
    const float own = e < k ? p.share[t * k + e] : 0.f;
    float q = 0.f;
    bool first = true;
    for (int o0 = 0; o0 < k; o0 += 64) {
      const int mine = o0 + lane;
      const int32_t other = in_vocab(p, t * k + mine, mine < k);
      const float share = mine < k ? p.share[t * k + mine] : 0.f;
      const int n = k - o0 < 64 ? k - o0 : 64;
      for (int o = 0; o < n; ++o) {
        const bool same = __builtin_amdgcn_readlane(other, o) == id;
        const float more = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int32_t, share), o));
        q += same ? more : 0.f;
        first = first && !(same && more != 0.f && o0 + o < e);
      }
    }
    if (!here || !first || own == 0.f) continue;  // an id's first entry with a share places it: it has a product
    E* out = static_cast<E*>(p.grad) + i * p.vpiece + v;
    if constexpr (std::is_same_v<T, float>) {
      E* low = out + p.tpad * p.vpiece;
      split_f16((static_cast<float>(*out) + static_cast<float>(*low)) - b * q, *out, *low);
    } else {
      const float of_v = is_far(m2) ? to_f32(*out) : a * fast_exp2(fmaf(p.picked[t * k + e], c, -m2));
      *out = from_f32<E>(of_v - b * q);
    }
  }
}

// dhidden over a piece: m along the dim, n along the tokens, terms along the vocabulary.
template <typename T>
__global__ __launch_bounds__(512, 2) void loss_dhidden_kernel(const LossParams p, int64_t vp, bool add) {
  using E = Kept<T>;
  const int64_t kept = p.scal->kept;
  const int64_t mts = (p.dpad + kLossTile - 1) / kLossTile, nts = (kept + kLossTile - 1) / kLossTile;
  const int splits = p.scal->hsplit;
  int64_t mt, ns;
  if (!tile_of(p.first + blockIdx.x, mts, nts * splits, mt, ns)) return;
  const int64_t nt = ns / splits;
  const int split = static_cast<int>(ns - nt * splits);
  constexpr int runs = kRuns<T>;
  const ProductParams q = {weight_operand(p, vp), grad_operand(p), p.vrows, runs};
  const int depths = static_cast<int>(p.vrows / kLossDepth) * runs;
  MCPU_TILE_LDS(a0, b0, a1, b1);
  Acc acc;
  tile_product<E, true, false>(q, mt * kLossTile, nt * kLossTile, static_cast<int>(int64_t{depths} * split / splits),
                               static_cast<int>(int64_t{depths} * (split + 1) / splits), a0, b0, a1, b1, acc);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int64_t t = nt * kLossTile + (wave & 3) * 64 + j * 32 + (lane & 31);
    float* out = p.acc + (split * nts * kLossTile + t) * p.dpad;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int64_t d = mt * kLossTile + (wave >> 2) * 128 + 32 * i + 8 * g + 4 * (lane >> 5);
        if (d >= p.dpad) continue;
        float4 v = make_float4(acc.v[j][i][4 * g], acc.v[j][i][4 * g + 1], acc.v[j][i][4 * g + 2],
                               acc.v[j][i][4 * g + 3]);
        float4* to = reinterpret_cast<float4*>(out + d);
        if (add) {
          const float4 o = *to;
          v = make_float4(v.x + o.x, v.y + o.y, v.z + o.z, v.w + o.w);
        }
        *to = v;
      }
  }
}

// Sums of splits' results at four columns, eight loads on their way.
__device__ __forceinline__ void sum_splits(const float* at, int64_t stride, int splits, float (&v)[4]) {
  for (int s0 = 0; s0 < splits; s0 += 8) {
    float4 x[8];
#pragma unroll
    for (int u = 0; u < 8; ++u)
      x[u] = s0 + u < splits ? *reinterpret_cast<const float4*>(at + (s0 + u) * stride) : make_float4(0, 0, 0, 0);
#pragma unroll
    for (int u = 0; u < 8; ++u) v[0] += x[u].x, v[1] += x[u].y, v[2] += x[u].z, v[3] += x[u].w;
  }
}

// dhidden in its own type: the splits' sum; rows that do not count have none. A wave 256 columns of a row.
template <typename T> __global__ __launch_bounds__(256) void loss_dhidden_out_kernel(const LossParams p) {
  using E = Kept<T>;
  const int64_t at = (p.first + blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t across = (p.dim + 255) / 256, i = at / across, d = (at - i * across) * 256 + (threadIdx.x & 63) * 4;
  if (i >= p.tokens || d >= p.dim) return;
  const bool in = i < p.scal->kept;
  float v[4] = {};
  if (in) {
    float scale = unit_of<E>(p, i) / kUp<E>;
    if constexpr (std::is_same_v<T, float>) scale *= pow2(-up_exponent(p.scal->wmax));
    const int64_t rows = (int64_t{p.scal->kept} + kLossTile - 1) / kLossTile * kLossTile;
    sum_splits(p.acc + i * p.dpad + d, rows * p.dpad, p.scal->hsplit, v);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] *= scale;
  }
  st_upto4<T>(static_cast<T*>(p.dhidden) + p.rows[i] * p.dim, d, upto4(p.dim - d), v);
}

// dweight of a piece: m along the dim, n along the vocabulary, terms along the tokens.
template <typename T>
__global__ __launch_bounds__(512, 2) void loss_dweight_kernel(const LossParams p, int64_t vp) {
  using E = Kept<T>;
  const int64_t mts = (p.dpad + kLossTile - 1) / kLossTile;
  int64_t mt, ns;
  if (!tile_of(p.first + blockIdx.x, mts, p.vrows / kLossTile * p.wsplit, mt, ns)) return;
  const int64_t nt = ns / p.wsplit;
  const int split = static_cast<int>(ns - nt * p.wsplit);
  constexpr int runs = kRuns<T>;
  const int64_t depth = (int64_t{p.scal->kept} + kLossDepth - 1) / kLossDepth * kLossDepth;
  const ProductParams q = {rows_operand(p, p.hscaled != nullptr ? p.hscaled : p.hrows), grad_operand(p), depth, runs};
  const int depths = static_cast<int>(depth / kLossDepth) * runs;
  MCPU_TILE_LDS(a0, b0, a1, b1);
  Acc acc;
  tile_product<E, true, true>(q, mt * kLossTile, nt * kLossTile,
                              static_cast<int>(int64_t{depths} * split / p.wsplit),
                              static_cast<int>(int64_t{depths} * (split + 1) / p.wsplit), a0, b0, a1, b1, acc);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const float scale = p.scal->unit / kUp<E> * pow2(-dweight_exponent<T>(p));
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int64_t vl = nt * kLossTile + (wave & 3) * 64 + j * 32 + (lane & 31);
    const int64_t v = vp + vl;
    if (v >= p.vocab) continue;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int64_t d = mt * kLossTile + (wave >> 2) * 128 + 32 * i + 8 * g + 4 * (lane >> 5);
        if (d >= p.dim) continue;
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = acc.v[j][i][4 * g + e] * scale;
        if (p.dwpart != nullptr)
          *reinterpret_cast<float4*>(p.dwpart + (split * p.vpiece + vl) * p.dpad + d) =
              make_float4(x[0], x[1], x[2], x[3]);
        else
          st_upto4<T>(static_cast<T*>(p.dweight) + v * p.dim, d, upto4(p.dim - d), x);
      }
  }
}

// dweight of a piece from its splits. A wave 256 columns of a row.
template <typename T> __global__ __launch_bounds__(256) void loss_dweight_out_kernel(const LossParams p, int64_t vp) {
  const int64_t at = (p.first + blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t across = (p.dim + 255) / 256, vl = at / across;
  const int64_t d = (at - vl * across) * 256 + (threadIdx.x & 63) * 4;
  if (vl >= p.vrows || vp + vl >= p.vocab || d >= p.dim) return;
  float v[4] = {};
  sum_splits(p.dwpart + vl * p.dpad + d, p.vpiece * p.dpad, p.wsplit, v);
  st_upto4<T>(static_cast<T*>(p.dweight) + (vp + vl) * p.dim, d, upto4(p.dim - d), v);
}

// ---- the loss of a row, and of all ------------------------------------------------------------

// The loss of row t, the i-th that counts, from the maximum of its logits and the sum relative to it; cross
// entropy: of all but the target's, which comes by itself.
__device__ __forceinline__ void finish_row(const LossParams& p, int64_t t, int64_t i, float top, float sum,
                                           float own) {
  const float c = kLog2e / p.temperature;
  float* stat = p.stat + i;
  if (p.teacher == nullptr) {
    // The target joins the others: relative to their maximum, as long as that is in float32's range.
    const float d = own - top;
    const bool far = !(d <= 40.f);
    // An overflowed target: lse - s is inf - inf, and the gradient NaN likewise.
    const float mine = own == INFINITY ? NAN : far ? 1.f : fast_exp2(d * c);
    const float others = far ? sum * fast_exp2(-d * c) : sum;
    const float all = mine + others;
    // log(all / mine), by log1p where the target is the largest.
    const float r = others / mine, u = 1.f + r;
    p.each[t] = d >= 0.f ? (u == 1.f ? r : logf(u) * (r / (u - 1.f))) : logf(all) - d;
    stat[2 * p.tokens] = mine / all;
    stat[3 * p.tokens] = others / all;
    top = far ? own : top;
    sum = all;
  }
  const float lse = top / p.temperature + logf(sum);
  p.lse[t] = lse;
  stat[0] = top;
  stat[p.tokens] = sum;
  if (p.teacher != nullptr) p.each[t] = (p.cross[t] + lse) * p.temperature * p.temperature;
}

// A thread's parts of one token, `step` apart: their maximum m and the sum s relative to it, eight loads on their way.
__device__ __forceinline__ void join_parts(const float2* part, int64_t stride, int64_t first, int step, int64_t parts,
                                           float c, float& m, float& s) {
  for (int64_t q0 = first; q0 < parts; q0 += step * 8) {
    float2 x[8];
    float top = m;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      x[u] = q0 + u * step < parts ? part[(q0 + u * step) * stride] : make_float2(-INFINITY, 0.f);
      top = fmaxf(top, x[u].x);
    }
    const float sub = top == -INFINITY ? 0.f : top;
    s *= fast_exp2((m - sub) * c);
#pragma unroll
    for (int u = 0; u < 8; ++u) s = fmaf(x[u].y, fast_exp2((x[u].x - sub) * c), s);
    m = top;
  }
}

// 32 tokens a workgroup: 32 threads a token join the parts, one takes the loss.
__global__ __launch_bounds__(1024) void loss_join_kernel(const LossParams p) {
  __shared__ float ms[32][33], ss[32][33];
  const int64_t kept = p.scal->kept;
  const int64_t i = (p.first + blockIdx.x) * 32 + (threadIdx.x & 31);
  const int slice = threadIdx.x >> 5;
  const int64_t parts = (p.vocab + kLossPart - 1) / kLossPart;
  const float c = kLog2e / p.temperature;
  float m = -INFINITY, s = 0.f;
  if (i < kept) join_parts(p.part + i, p.tpad, slice, 32, parts, c, m, s);
  ms[slice][threadIdx.x & 31] = m;
  ss[slice][threadIdx.x & 31] = s;
  __syncthreads();
  if (slice != 0 || i >= p.tokens) return;
  const int64_t t = p.rows[i];
  if (i >= kept) {
    p.lse[t] = 0.f;
    p.each[t] = 0.f;
    return;
  }
  const int x = threadIdx.x;
  float top = ms[0][x];
  for (int q = 1; q < 32; ++q) top = fmaxf(top, ms[q][x]);
  const float sub = top == -INFINITY ? 0.f : top;
  float sum = 0.f;
  for (int q = 0; q < 32; ++q) sum = fmaf(ss[q][x], fast_exp2((ms[q][x] - sub) * c), sum);
  finish_row(p, t, i, top, sum, p.teacher == nullptr ? p.picked[i] : 0.f);
}

// ---- few tokens, and blocks --------------------------------------------------------------------------

// Up to 64 tokens a workgroup, past which 128 vocabulary rows stream, 32 a wave. With
// 64 in all every row is read once, and what bounds it is HBM. A lane's part of an operand is row
// l % 16 and the 16 bytes at l / 16 of each 64, the same terms for both operands.
// float32 goes through v_mfma_f32_16x16x4_f32, four to 16 bytes.
typedef uint32_t u32x4_e2 __attribute__((ext_vector_type(4), aligned(2)));

template <typename T> constexpr int kChunk = 16 / static_cast<int>(sizeof(T));

template <typename T> __device__ __forceinline__ u32x4 chunk_at(const T* row, int64_t k) {
  return *reinterpret_cast<const u32x4_e2*>(row + k);
}
// A chunk of which the row may have less, or nothing.
template <typename T> __device__ __forceinline__ u32x4 chunk_left(const T* row, int64_t k, int64_t dim) {
  if (k + kChunk<T> <= dim) return chunk_at<T>(row, k);
  T v[kChunk<T>];
#pragma unroll
  for (int e = 0; e < kChunk<T>; ++e) v[e] = k + e < dim ? row[k + e] : T{};
  return __builtin_bit_cast(u32x4, v);
}
template <typename T> __device__ __forceinline__ f32x4 mma16(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (std::is_same_v<T, bf16>) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
  } else if constexpr (std::is_same_v<T, f16>) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                  0);
  } else {
    const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], y[e], c, 0, 0, 0);
    return c;
  }
}

// A stage of LDS: 128 bytes of each row of the workgroup's 128 of weight and NF x 16 of
// hidden. Three, 72 KiB at most, leave room for two workgroups on a CU; a fourth,
// where it leaves one, is 6 % slower, else as fast.
template <int NF> constexpr int kStageBytes = (128 + NF * 16) * 128;

// Products of whole groups of 128 bytes, where rows are 16-byte aligned: loads write
// straight into LDS, eight lanes a row of 128 bytes, in the order that spreads a read
// over the banks (chunk c of row r at c ^ (r % 8)). Straight into the operands'
// registers a load touches 16 rows, and the cache takes 50 cycles for it: 49 against
// 15 us with 3 tokens, 688 x 2560 bf16, and 70 against 59, 16 x 50280 x 2560 (257 MB).
template <typename T, int NF, typename Row>
__device__ __forceinline__ int64_t few_products_lds(const LossParams& p, Row&& row, int64_t v0,
                                                    f32x4 (&acc)[2][2][NF]) {
  constexpr int kHidden = NF > 2 ? 2 : 1, kLoads = 4 + kHidden;
  constexpr int kTerms = 128 / static_cast<int>(sizeof(T));
  __shared__ __attribute__((aligned(1024))) char s0[kStageBytes<NF>];
  __shared__ __attribute__((aligned(1024))) char s1[kStageBytes<NF>];
  __shared__ __attribute__((aligned(1024))) char s2[kStageBytes<NF>];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int groups = static_cast<int>(p.dim / kTerms);
  if (groups == 0) return 0;
  // A lane's 16 bytes of eight rows a load: four loads of the wave's own rows of
  // weight, and its share of hidden's (of 16 tokens, and of the last 16 of 48, waves 2 and 3 bring what 0 and 1 do).
  const int r8 = lane >> 3, swap = ((lane & 7) ^ r8) * (16 / static_cast<int>(sizeof(T)));
  const T* from[kLoads];
  int to[kLoads];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t v = v0 + 8 * i + r8;  // a row that is not there is read as the last
    from[i] = static_cast<const T*>(p.weight) + (v < p.vocab ? v : p.vocab - 1) * p.sw + swap;
    to[i] = (wave * 32 + 8 * i) * 128;
  }
#pragma unroll
  for (int i = 0; i < kHidden; ++i) {
    const int t8 = NF == 1 ? wave & 1 : NF == 3 && i == 1 ? 4 + (wave & 1) : wave + 4 * i;
    from[4 + i] = row(8 * t8 + r8) + swap;
    to[4 + i] = (128 + 8 * t8) * 128;
  }
  using lds_ptr = __attribute__((address_space(3))) void*;
  using global_ptr = const __attribute__((address_space(1))) void*;
  auto load = [&](char* stage, int group) {
    const int64_t at = int64_t{group < groups ? group : groups - 1} * kTerms;  // behind the end: once more, unused
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      __builtin_amdgcn_global_load_lds((global_ptr)(from[i] + at), (lds_ptr)(stage + to[i]), 16, 0, 0);
  };
  auto step = [&](const char* stage, char* next, int group) {
    // The loads of this group have arrived, those of the next need not have; and no wave reads `next` any more.
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0070 | kLoads);  // vmcnt(kLoads) lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    load(next, group + 2);
    __builtin_amdgcn_sched_barrier(0);
    const int r = lane & 15;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int at = ((u * 4 + (lane >> 4)) ^ (r & 7)) * 16;
      u32x4 a[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) a[i] = *reinterpret_cast<const u32x4*>(stage + (wave * 32 + 16 * i + r) * 128 + at);
#pragma unroll
      for (int j = 0; j < NF; ++j) {
        const u32x4 b = *reinterpret_cast<const u32x4*>(stage + (128 + 16 * j + r) * 128 + at);
#pragma unroll
        for (int i = 0; i < 2; ++i) acc[u][i][j] = mma16<T>(a[i], b, acc[u][i][j]);
      }
    }
  };
  load(s0, 0);
  load(s1, 1);
  int g = 0;
  for (; g + 3 <= groups; g += 3) {
    step(s0, s2, g);
    step(s1, s0, g + 1);
    step(s2, s1, g + 2);
  }
  if (g < groups) step(s0, s2, g);
  if (g + 1 < groups) step(s1, s0, g + 1);
  __builtin_amdgcn_s_waitcnt(0x0070);  // nothing is on its way into LDS any more
  return int64_t{groups} * kTerms;
}

// The products of NF x 16 rows of hidden and a wave's 32 rows of weight from v0 on:
// s[i][j][e] is of vocabulary row v0 + 16 i + 4 (lane / 16) + e and token 16 j + lane % 16;
// row(t) is where token t's row of hidden begins. Forward and backward form them alike,
// to the bit.
template <typename T, int NF, typename Row>
__device__ __forceinline__ void few_products(const LossParams& p, Row&& row, int64_t v0, f32x4 (&s)[2][NF]) {
  const int lane = threadIdx.x & 63;
  const int64_t k0 = (lane >> 4) * kChunk<T>;
  // Two sums of every other load's products: half the roundings in a row.
  f32x4 acc[2][2][NF];
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < NF; ++j) acc[u][i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  int64_t k = p.few_lds ? few_products_lds<T, NF>(p, row, v0, acc) : 0;
  // Rows that are not aligned, and what is left of those that are: into registers, two loads a turn.
  const T *w[2], *h[NF];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int64_t v = v0 + 16 * i + (lane & 15);  // a row that is not there is read as the last
    w[i] = static_cast<const T*>(p.weight) + (v < p.vocab ? v : p.vocab - 1) * p.sw;
  }
#pragma unroll
  for (int j = 0; j < NF; ++j) h[j] = row(16 * j + (lane & 15));
  constexpr int kStep = 4 * kChunk<T>;  // terms of a load
  for (; k + 2 * kStep <= p.dim; k += 2 * kStep) {
    u32x4 a[2][2], b[2][NF];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int i = 0; i < 2; ++i) a[u][i] = chunk_at<T>(w[i], k + k0 + u * kStep);
#pragma unroll
      for (int j = 0; j < NF; ++j) b[u][j] = chunk_at<T>(h[j], k + k0 + u * kStep);
    }
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < NF; ++j) acc[u][i][j] = mma16<T>(a[u][i], b[u][j], acc[u][i][j]);
  }
  for (; k < p.dim; k += kStep) {
    u32x4 x[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) x[i] = chunk_left<T>(w[i], k + k0, p.dim);
#pragma unroll
    for (int j = 0; j < NF; ++j) {
      const u32x4 y = chunk_left<T>(h[j], k + k0, p.dim);
#pragma unroll
      for (int i = 0; i < 2; ++i) acc[0][i][j] = mma16<T>(x[i], y, acc[0][i][j]);
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < NF; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[i][j][e] = acc[0][i][j][e] + acc[1][i][j][e];
}

// Tokens that a row of parts of NF groups has room for: 16, 32 or 64.
constexpr int few_wide(int groups) { return groups > 2 ? 64 : groups * 16; }

// NF x 16 tokens and 128 vocabulary rows a workgroup, and of these one maximum and sum a token.
// Up to 64 tokens in all (not ROWS), as they come; distillation: one more workgroup a
// token, first, for the teacher's part, which would take 10 us before or after.
// ROWS: 64 of the rows that count a workgroup, as loss_logits_kernel takes and leaves
// them, where its tiles are too few to fill the GPU.
template <typename T, int NF, bool ROWS>
__global__ __launch_bounds__(256, 2) void loss_few_kernel(const LossParams p) {
  const int64_t teachers = !ROWS && p.teacher != nullptr ? p.tokens : 0;
  const int64_t at = p.first + blockIdx.x - teachers;
  if (at < 0) return teacher_row<T, 256>(p, at + teachers);
  const int64_t groups = (p.vocab + kLossPart - 1) / kLossPart;
  const int64_t group = ROWS ? at % groups : at, t0 = ROWS ? at / groups * kLossFew : 0;
  const int64_t tokens = ROWS ? p.scal->kept : p.tokens;
  if (t0 >= tokens) return;
  __shared__ float2 parts[4][NF * 16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t v0 = group * kLossPart + wave * 32;
  auto row = [&](int64_t t) { return ROWS ? int64_t{p.rows[t]} : t; };
  f32x4 acc[2][NF];
  few_products<T, NF>(p, [&](int64_t i) {  // a token that is not there is read as the last
    return static_cast<const T*>(p.hidden) + row(t0 + i < tokens ? t0 + i : tokens - 1) * p.sh;
  }, v0, acc);
  const float c = kLog2e / p.temperature;
#pragma unroll
  for (int j = 0; j < NF; ++j) {
    const int64_t t = t0 + 16 * j + (lane & 15);
    const bool aim = p.teacher == nullptr && t < tokens && (ROWS || counts(p, t));
    const int64_t target = aim ? id_at(p, row(t)) : -1;
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int64_t v = v0 + 16 * i + 4 * (lane >> 4) + e;
        if (v == target) p.picked[t] = acc[i][j][e];
        if (v == target || v >= p.vocab) acc[i][j][e] = -INFINITY;
        m = fmaxf(m, acc[i][j][e]);
      }
    m = fmaxf(m, __shfl_xor(m, 16));
    m = fmaxf(m, __shfl_xor(m, 32));
    const float sub = m == -INFINITY ? 0.f : m;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) s += fast_exp2((acc[i][j][e] - sub) * c);
    s += __shfl_xor(s, 16);
    s += __shfl_xor(s, 32);
    if (lane < 16) parts[wave][16 * j + lane] = make_float2(m, s);
  }
  __syncthreads();
  const int i = threadIdx.x;
  if (i >= NF * 16 || t0 + i >= tokens) return;
  float m = parts[0][i].x, s = 0.f;
  for (int q = 1; q < 4; ++q) m = fmaxf(m, parts[q][i].x);
  const float sub = m == -INFINITY ? 0.f : m;
  for (int q = 0; q < 4; ++q) s = fmaf(parts[q][i].y, fast_exp2((parts[q][i].x - sub) * c), s);
  p.part[group * (ROWS ? p.tpad : few_wide(NF)) + t0 + i] = make_float2(m, s);
}

// ds of 64 of the rows that count a workgroup, as loss_grad_kernel; rows behind the last, up to whole 64, are zero.
template <typename T, int NF>
__global__ __launch_bounds__(256, 2) void loss_few_grad_kernel(const LossParams p, int64_t vp) {
  using E = Kept<T>;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t at = p.first + blockIdx.x, groups = p.vrows / kLossPart, t0 = at / groups * kLossFew;
  const int64_t vl = at % groups * kLossPart + wave * 32, v0 = vp + vl;
  const int64_t kept = p.scal->kept;
  if (t0 >= kept) return;
  f32x4 acc[2][NF];
  few_products<T, NF>(p, [&](int64_t i) {
    return static_cast<const T*>(p.hidden) + p.rows[t0 + i < kept ? t0 + i : kept - 1] * p.sh;
  }, v0, acc);
  const float c = kLog2e / p.temperature;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int64_t t = t0 + 16 * j + (lane & 15);
    const bool in = j < NF && t < kept;
    const float up = in ? kUp<E> / unit_of<E>(p, t) : 0.f;
    const float a = in ? p.coef[t] * up : 0.f, b = in ? p.coef[p.tpad + t] * up : 0.f;
    const float m2 = in ? p.coef[2 * p.tpad + t] : 0.f, top = in ? p.stat[t] : 0.f;
    const int64_t target = in && p.target != nullptr ? p.target[t] : -1;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int64_t at = 16 * i + 4 * (lane >> 4);
      float x[4] = {};
      if (in) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int64_t v = v0 + at + e;
          const float s = acc[i][j < NF ? j : 0][e], power = is_far(m2) ? (s - top) * c : fmaf(s, c, -m2);
          x[e] = v >= p.vocab ? 0.f : v == target ? b : a * fast_exp2(power);
        }
      }
      E* out = static_cast<E*>(p.grad) + t * p.vpiece + vl + at;
      st4_elem<E>(out, 0, x);
      if constexpr (std::is_same_v<T, float>) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          f16 hi, lo;
          split_f16(x[e], hi, lo);
          x[e] = static_cast<float>(lo);
        }
        st4_elem<E>(out, p.tpad * p.vpiece, x);
      }
    }
  }
}

// As f<16-token groups>() for up to 64 tokens. 33 tokens as three groups, not four: 148 against 185 us for
// 50280 x 2560 float32, 64 against 65.5 in bf16.
template <typename F> void for_few(int64_t tokens, F&& f) {
  if (tokens <= 16)
    f(std::integral_constant<int, 1>{});
  else if (tokens <= 32)
    f(std::integral_constant<int, 2>{});
  else if (tokens <= 48)
    f(std::integral_constant<int, 3>{});
  else
    f(std::integral_constant<int, 4>{});
}

// The rows that count, their losses and all rows' of up to kWide tokens: one workgroup. A wave reads 512 bytes of
// parts at a time, a token to every kWide lanes: 7.3 us for 33 tokens and 393 parts, 9.6 with 32 bytes of a
// token to each 16 threads.
template <int kWide> __global__ __launch_bounds__(1024) void loss_few_join_kernel(const LossParams p) {
  constexpr int kSlices = 1024 / kWide;
  const int n = static_cast<int>(p.tokens);
  __shared__ float2 sums[kSlices][kWide + 1];
  __shared__ float losses[64];
  __shared__ unsigned long long mask;
  if (threadIdx.x < 64) {
    const unsigned long long m = __ballot(threadIdx.x < n && counts(p, threadIdx.x));
    if (threadIdx.x == 0) mask = m;
    losses[threadIdx.x] = 0.f;
  }
  const int64_t parts = (p.vocab + kLossPart - 1) / kLossPart;
  const float c = kLog2e / p.temperature;
  {
    const int t = threadIdx.x % kWide, slice = threadIdx.x / kWide;
    float m = -INFINITY, s = 0.f;
    if (t < n) join_parts(p.part + t, kWide, slice, kSlices, parts, c, m, s);
    sums[slice][t] = make_float2(m, s);
  }
  __syncthreads();
  // 16 threads a token.
  const int t = threadIdx.x >> 4, j = threadIdx.x & 15;
  const bool keep = mask >> t & 1;
  const int kept = __popcll(mask), before = __popcll(mask & ((1ull << t) - 1));
  if (t < n) {
    float m = -INFINITY, s = 0.f;
#pragma unroll
    for (int q = j; q < kSlices; q += 16) m = fmaxf(m, sums[q][t].x);
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) m = fmaxf(m, __shfl_xor(m, o));
    const float sub = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int q = j; q < kSlices; q += 16) s = fmaf(sums[q][t].y, fast_exp2((sums[q][t].x - sub) * c), s);
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) s += __shfl_xor(s, o);
    if (j == 0) {
      if (keep) {
        finish_row(p, t, before, m, s, p.teacher == nullptr ? p.picked[t] : 0.f);
      } else {
        p.lse[t] = 0.f;
        p.each[t] = 0.f;
      }
      p.rows[keep ? before : kept + t - before] = t;
      losses[t] = p.each[t];
      if (t == 0) p.rows[n] = kept;
    }
  }
  if (p.reduction == MCPU_REDUCE_NONE) return;
  __syncthreads();
  if (threadIdx.x >= 64) return;
  float sum = losses[threadIdx.x];
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) sum += __shfl_xor(sum, o);
  if (threadIdx.x == 0)
    p.loss[0] = p.reduction == MCPU_REDUCE_MEAN ? sum / static_cast<float>(kept > 0 ? kept : 1) : sum;
}

// ---- all rows ------------------------------------------------------------------------------------

// The sum or mean of the rows' losses, one workgroup, in a fixed order.
__global__ __launch_bounds__(1024) void loss_sum_kernel(const LossParams p) {
  __shared__ float sums[16];
  float s = 0.f, lost = 0.f;  // compensated
  for (int64_t t = threadIdx.x; t < p.tokens; t += 1024) {
    const float y = p.each[t] - lost, next = s + y;
    lost = (next - s) - y;
    s = next;
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) s += __shfl_xor(s, o);
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x != 0) return;
  s = 0.f;
  for (int i = 0; i < 16; ++i) s += sums[i];
  const int32_t kept = p.scal->kept;
  p.loss[0] = p.reduction == MCPU_REDUCE_MEAN ? s / static_cast<float>(kept > 0 ? kept : 1) : s;
}

// Coefficients of the rows that count, and the unit each one's ds is kept in. In
// 16 bits a rounding of the target's ds, the row's largest, would be in all of
// the row's gradient alike; so the unit is that ds itself (exactly 1 then), and
// dweight takes the units from hidden's rows, scaled by unit / the largest unit.
// Distillation has no one largest: one unit, the largest coefficient; f16 pieces
// with a gradient for each row: that row's coefficient, down to a power of two, which
// rounds nothing of hidden. One workgroup.
__global__ __launch_bounds__(1024) void loss_coef_kernel(const LossParams p) {
  __shared__ float tops[16], largest[16];
  const int32_t kept = p.rows[p.tokens];
  const float share = p.reduction == MCPU_REDUCE_MEAN ? 1.f / static_cast<float>(kept > 0 ? kept : 1) : 1.f;
  const float c = kLog2e / p.temperature;
  const bool each = p.reduction == MCPU_REDUCE_NONE;
  const float all = each ? 0.f : p.dloss[0] * share;
  // By the rows that count, which the host does not know; beside the others' loads.
  if (threadIdx.x == 1023)
    p.scal->hsplit = splits_for((p.dpad + kLossTile - 1) / kLossTile * ((kept + kLossTile - 1) / kLossTile),
                                p.vpiece / kLossDepth * (p.dtype == MCPU_F32 ? 3 : 1), true);
  float most = 0.f, factor = 0.f;  // the largest unit, and the largest softmax coefficient
  for (int64_t i0 = threadIdx.x; i0 < kept; i0 += 1024 * 8) {
    float g[8], e[8], stat[4][8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int64_t i = i0 + u * 1024 < kept ? i0 + u * 1024 : i0;
      const int64_t t = each || p.dlse != nullptr ? p.rows[i] : 0;
      g[u] = !each ? all : p.dloss != nullptr ? p.dloss[t] : 0.f;
      e[u] = p.dlse != nullptr ? p.dlse[t] : 0.f;
#pragma unroll
      for (int q = 0; q < 4; ++q) stat[q][u] = q < 2 || p.share == nullptr ? p.stat[q * p.tokens + i] : 0.f;
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int64_t i = i0 + u * 1024;
      if (i >= kept) break;
      g[u] *= p.temperature;  // 1 for cross entropy
      const float a = g[u] + e[u];
      // exp(c (s - maximum)) as 2^(c s - m2), with the rounding of m2 in the factor.
      const float m2 = stat[0][u] * c, off = is_far(m2) ? 0.f : fmaf(stat[0][u], c, -m2);
      // Cross entropy: the target's ds, a p - g = (a - g) p - g (1 - p); no other is above a (1 - p).
      const float own = p.share != nullptr ? g[u] : e[u] * stat[2][u] - g[u] * stat[3][u];
      const float top = fmaxf(__builtin_fabsf(own), __builtin_fabsf(a) * (p.share != nullptr ? 1.f : stat[3][u]));
      if (top < INFINITY) most = fmaxf(most, top);
      if (__builtin_fabsf(a) < INFINITY) factor = fmaxf(factor, __builtin_fabsf(a));
      p.coef[i] = a / stat[1][u] * fmaf(-kLn2, off, 1.f);
      p.coef[p.tpad + i] = own;
      p.coef[2 * p.tpad + i] = m2;
      // Not where a / unit would leave float32's range: the others' share is below 2^-90, a loss of 0 but for that.
      const bool fits = top > 0x1p-100f && top > __builtin_fabsf(a) * 0x1p-90f && top < INFINITY;
      p.coef[3 * p.tpad + i] = fits && p.hscaled != nullptr ? (p.share == nullptr ? top : power_below(top)) : 0.f;
    }
  }
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) {
    most = fmaxf(most, __shfl_xor(most, s));
    factor = fmaxf(factor, __shfl_xor(factor, s));
  }
  if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = most, largest[threadIdx.x >> 6] = factor;
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int i = 1; i < 16; ++i) most = fmaxf(most, tops[i]), factor = fmaxf(factor, largest[i]);
  most = fmaxf(most, factor * 0x1p-90f);
  p.scal->kept = kept;
  p.scal->hmax = 0;
  p.scal->wmax = p.laid != nullptr ? *p.laid : 0;
  most = most == 0.f ? 1.f : fmaxf(most, 0x1p-100f);
  p.scal->unit = p.share != nullptr && p.hscaled != nullptr ? power_below(most) : most;
}

// Results of calls without rows, vocabulary or entries.
__global__ __launch_bounds__(256) void loss_zero_kernel(uint8_t* at, int64_t bytes) {
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < bytes; i += 256ll * gridDim.x) at[i] = 0;
}

// ---- launches -----------------------------------------------------------------------------------

template <typename K, typename... A>
void run(K kernel, LossParams p, int64_t groups, int threads, hipStream_t st, A... more) {
  launch_all(groups, threads, [&](int64_t first, unsigned count) {
    p.first = first;
    hipLaunchKernelGGL(kernel, dim3(count), dim3(threads), 0, st, p, more...);
  });
}

template <typename T> void lay_operands(const LossParams& p, bool weight, hipStream_t st) {
  if constexpr (std::is_same_v<T, float>) {
    run(loss_most_kernel<T>, p, std::min<int64_t>((p.tokens + 15) / 16, 256), 1024, st, false);
    if (weight) run(loss_most_kernel<T>, p, std::min<int64_t>((p.vocab + 15) / 16, 256), 1024, st, true);
  } else if (std::is_same_v<T, f16> && p.hscaled != nullptr && p.dweight != nullptr) {
    run(loss_most_kernel<T>, p, std::min<int64_t>((p.tokens + 15) / 16, 256), 1024, st, false);
  }
  run(loss_gather_kernel<T>, p, p.tpad / 4, 256, st);
  if (weight && p.wrows != nullptr) run(loss_weight_kernel<T>, p, (p.vocab + 3) / 4, 256, st);
}

template <typename T> hipError_t fwd(const LossParams& p, hipStream_t st) {
  if (p.tokens <= kLossFew) {
    for_few(p.tokens, [&](auto nf) {
      run(loss_few_kernel<T, decltype(nf)::value, false>, p,
          (p.vocab + kLossPart - 1) / kLossPart + (p.teacher != nullptr ? p.tokens : 0), 256, st);
      run(loss_few_join_kernel<few_wide(decltype(nf)::value)>, p, 1, 1024, st);
    });
    return hipGetLastError();
  }
  if (p.teacher != nullptr) run(loss_teacher_kernel<T>, p, p.tokens, 256, st);
  run(loss_rows_kernel, p, 1, 1024, st);
  if (p.blocks) {
    run(loss_few_kernel<T, 4, true>, p,
        (p.vocab + kLossPart - 1) / kLossPart * ((p.tokens + kLossFew - 1) / kLossFew), 256, st);
  } else {
    lay_operands<T>(p, true, st);
    run(loss_logits_kernel<T>, p, (p.vocab + kLossTile - 1) / kLossTile * (p.tpad / kLossTile), 512, st);
  }
  run(loss_join_kernel, p, (p.tokens + 31) / 32, 1024, st);
  if (p.reduction != MCPU_REDUCE_NONE) run(loss_sum_kernel, p, 1, 1024, st);
  return hipGetLastError();
}

template <typename T> hipError_t bwd(LossParams p, hipStream_t st) {
  run(loss_coef_kernel, p, 1, 1024, st);
  // Blocks of 64 tokens read weight as it lies.
  lay_operands<T>(p, p.laid == nullptr && (!p.blocks || p.dhidden != nullptr), st);
  const int64_t tt = p.tpad / kLossTile, dt = (p.dpad + kLossTile - 1) / kLossTile;
  float* const dwpart = p.dwpart;
  for (int64_t vp = 0; vp < p.vocab; vp += p.vpiece) {
    p.vrows = loss_piece_rows(p, vp);
    const int64_t vt = p.vrows / kLossTile;
    if (p.blocks)
      for_few(p.tokens, [&](auto nf) {
        run(loss_few_grad_kernel<T, decltype(nf)::value>, p,
            p.vrows / kLossPart * ((p.tokens + kLossFew - 1) / kLossFew), 256, st, vp);
      });
    else
      run(loss_grad_kernel<T>, p, vt * tt, 512, st, vp);
    if (p.share != nullptr) run(loss_place_kernel<T>, p, (p.tokens + 3) / 4, 256, st, vp);
    if (p.dhidden != nullptr) run(loss_dhidden_kernel<T>, p, p.htiles, 512, st, vp, vp > 0);
    if (p.dweight != nullptr) {
      p.wsplit = loss_wsplit(p, vp);
      p.dwpart = p.wsplit > 1 ? dwpart : nullptr;
      run(loss_dweight_kernel<T>, p, dt * vt * p.wsplit, 512, st, vp);
      if (p.wsplit > 1) run(loss_dweight_out_kernel<T>, p, (p.vrows * ((p.dim + 255) / 256) + 3) / 4, 256, st, vp);
    }
  }
  if (p.dhidden != nullptr) run(loss_dhidden_out_kernel<T>, p, (p.tokens * ((p.dim + 255) / 256) + 3) / 4, 256, st);
  return hipGetLastError();
}

}  // namespace

// The way, the vocabulary piece and the splits. The piece: its ds is at most 1 GiB, and of the sizes below that
// give whole rounds of dweight's tiles, or equal pieces, the one that takes least.
// Twice as much would gain 1 % (16384 x 50280 x 768) to 3 % (32768), at 2560 columns nothing.
void loss_plan(LossParams& p) {
  const int pieces = loss_pieces(p.dtype), runs = pieces == 2 ? 3 : 1;
  auto up = [](int64_t n, int64_t to) { return (n + to - 1) / to; };
  p.tpad = up(p.tokens, kLossTile) * kLossTile;
  p.dpad = up(p.dim, kLossDepth) * kLossDepth;
  const int64_t all = up(p.vocab, kLossTile), tt = p.tpad / kLossTile, dt = up(p.dpad, kLossTile);
  const int64_t most = std::max<int64_t>(1, std::min(all, (int64_t{1} << 29) / pieces / p.tpad / kLossTile));
  const int64_t per = kLossTile / kLossDepth;  // depths of a tile's rows
  auto hsplit = [&](int64_t vt) { return splits_for(dt * tt, vt * per * runs, true); };
  auto piece = [&](int64_t n, int h) {
    const int w = splits_for(dt * n, tt * per * runs, false);
    return product_us<int64_t>(n * tt, p.dpad / kLossDepth * runs, 1, false) +
           product_us<int64_t>(dt * tt, n * per * runs, h, true) +
           product_us<int64_t>(dt * n, tt * per * runs, w, false) + 10;
  };
  auto cost = [&](int64_t vt) {
    const int h = hsplit(vt);
    const int64_t left = all % vt;
    return static_cast<float>(all / vt) * piece(vt, h) + (left > 0 ? piece(left, h) : 0.f);
  };
  int64_t best = up(all, up(all, most));  // equal pieces
  float least = cost(best);
  for (int64_t rounds = 1; rounds <= 8; ++rounds) {
    const int64_t vt = 256 * rounds / dt;
    if (vt < 1 || vt > most) continue;
    const float us = cost(vt);
    if (us < 0.99f * least) least = us, best = vt;
  }
  p.vpiece = best * kLossTile;
  // Blocks where all of them are on the GPU at once, two a CU: tiles of 256 x 256 would
  // be on an eighth of it to a quarter. Forward and backward, us: 512 x 4096 x 2560 bf16
  // 74 and 133 in tiles, 31 and 97 in blocks; 1024 x 8192 x 2560, twice what fits, 75 and
  // 194, 67 and 196; 256 x 50280 x 768 44 and 135, 71 and 175.
  p.blocks = p.tokens <= kLossFew || up(p.vocab, kLossPart) * up(p.tokens, kLossFew) <= kLossBlocks;
  p.htiles = std::max(dt * tt, std::min<int64_t>(kLossSplitTiles, kLossMostSplits * dt * tt));
  p.wsplit = std::max(loss_wsplit(p, 0), loss_wsplit(p, (all - 1) / best * p.vpiece));
}

int64_t loss_piece_rows(const LossParams& p, int64_t vp) {
  const int64_t left = (p.vocab - vp + kLossTile - 1) / kLossTile * kLossTile;
  return std::min(left, p.vpiece);
}
int loss_wsplit(const LossParams& p, int64_t vp) {
  const int64_t dt = (p.dpad + kLossTile - 1) / kLossTile;
  return splits_for(dt * (loss_piece_rows(p, vp) / kLossTile),
                    p.tpad / kLossDepth * (loss_pieces(p.dtype) == 2 ? 3 : 1), false);
}

hipError_t loss_zero(void* at, int64_t bytes, hipStream_t st) {
  if (bytes <= 0) return hipSuccess;
  hipLaunchKernelGGL(loss_zero_kernel, dim3(static_cast<unsigned>(std::min<int64_t>((bytes + 255) / 256, 4096))),
                     dim3(256), 0, st, static_cast<uint8_t*>(at), bytes);
  return hipGetLastError();
}

hipError_t loss_fwd_launch(LossParams p, hipStream_t st) {
  if (p.dtype == MCPU_F32) return fwd<float>(p, st);
  return p.dtype == MCPU_BF16 ? fwd<bf16>(p, st) : fwd<f16>(p, st);
}

hipError_t loss_bwd_launch(LossParams p, hipStream_t st) {
  if (p.dtype == MCPU_F32) return bwd<float>(p, st);
  return p.dtype == MCPU_BF16 ? bwd<bf16>(p, st) : bwd<f16>(p, st);
}

}  // namespace mcpu
