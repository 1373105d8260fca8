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
// Forward: rows that count are gathered, then one product whose epilogue keeps
// a maximum and a sum of 128 vocabulary rows per token, then one pass that joins
// these. A target's logit is taken from the product; the products of hidden with a
// teacher's ids are formed by themselves.
// Backward: a piece of the vocabulary at a time, the product again, now with ds in
// 16 bits as its result (float32: two f16 pieces), the ids' places put right, and
// the two products of the gradients over it. Rows that do not count take part in
// no product, so nothing in them, NaN included, reaches another row.
//
// Everything is summed in float32 in an order that depends on the sizes alone.
#include "launch.h"
#include "lm_math.h"
#include "tile_product.h"

namespace mcpu {
namespace {

// ds is kept as ds / unit times this: f16 then resolves 2^-37 of the largest coefficient.
template <typename E> constexpr float kUp = std::is_same_v<E, bf16> ? 1.f : 8192.f;

__device__ __forceinline__ int64_t id_at(const LossParams& p, int64_t i) {
  return p.ids64 ? static_cast<const int64_t*>(p.ids)[i] : static_cast<const int32_t*>(p.ids)[i];
}

// The power of two that brings a largest magnitude (as bits) to [2^13, 2^14), and its inverse.
__device__ __forceinline__ int up_exponent(uint32_t most) {
  if (most == 0) return 0;
  const int e = 13 - (static_cast<int>(most >> 23) - 127);
  return e > 120 ? 120 : e;
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

// Distillation: a wave a token.
template <typename T> __global__ __launch_bounds__(256) void loss_teacher_kernel(const LossParams p) {
  const int lane = threadIdx.x & 63;
  const int64_t t = (p.first + blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (t >= p.tokens) return;
  const int k = static_cast<int>(p.k);
  const float* teacher = p.teacher + t * k;
  float* share = p.share + t * k;
  const float c = 1.f / p.temperature;
  auto in = [&](int i) {
    const int64_t id = id_at(p, t * k + i);
    return id >= 0 && id < p.vocab;
  };
  // An entry of -inf has no share; NaN has, and makes the row NaN.
  float m = -INFINITY;
  bool any = false;
  for (int i = lane; i < k; i += 64)
    if (in(i) && !(teacher[i] == -INFINITY)) {
      any = true;
      m = fmaxf(m, teacher[i]);
    }
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) m = fmaxf(m, __shfl_xor(m, s));
  const bool keep = __any(any);
  float sum = 0.f;
  for (int i = lane; i < k; i += 64)
    if (in(i) && !(teacher[i] == -INFINITY)) sum += exp_acc((teacher[i] - m) * c);
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) sum += __shfl_xor(sum, s);
  const float logsum = logf(sum), inv = 1.f / sum;
  for (int i = lane; i < k; i += 64)
    share[i] = in(i) && !(teacher[i] == -INFINITY) ? exp_acc((teacher[i] - m) * c) * inv : 0.f;
  // The products, 16 lanes each, and sum q (log q - c s).
  const int j = lane & 15;
  float cross = 0.f;
  for (int i = lane >> 4; i < k; i += 4) {
    const bool have = in(i) && !(teacher[i] == -INFINITY);
    float s = 0.f;
    if (have)
      s = dot16<T>(static_cast<const T*>(p.hidden) + t * p.sh,
                   static_cast<const T*>(p.weight) + id_at(p, t * k + i) * p.sw, p.dim, j);
    if (j == 0) p.picked[t * k + i] = s;
    if (have) {
      const float x = (teacher[i] - m) * c, q = exp_acc(x) * inv;
      if (!(q == 0.f)) cross = fmaf(q, (x - logsum) - c * s, cross);
    }
  }
  cross += __shfl_xor(cross, 16);
  cross += __shfl_xor(cross, 32);
  if (lane == 0) {
    p.keep[t] = keep;
    p.cross[t] = cross;
  }
}

__device__ __forceinline__ bool counts(const LossParams& p, int64_t t) {
  if (p.teacher != nullptr) return p.keep[t];
  const int64_t id = id_at(p, t);
  return id >= 0 && id < p.vocab && id != p.ignore;
}

// The rows that count, in order, then the others; one workgroup, 16 rows a thread at a time.
__global__ __launch_bounds__(1024) void loss_rows_kernel(const LossParams p) {
  __shared__ int32_t sums[16];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int64_t kept = 0;
  for (int64_t t0 = 0; t0 < p.tokens; t0 += 16384) {
    const int64_t lo = t0 + threadIdx.x * 16;
    uint32_t mask = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (lo + i < p.tokens) mask |= static_cast<uint32_t>(counts(p, lo + i)) << i;
    const int32_t n = __popc(mask);
    int32_t before = n;
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
      const int32_t o = __shfl_up(before, s);
      if (lane >= s) before += o;
    }
    if (lane == 63) sums[w] = before;
    __syncthreads();
    int32_t base = 0, all = 0;
    for (int i = 0; i < 16; ++i) {
      base += i < w ? sums[i] : 0;
      all += sums[i];
    }
    __syncthreads();
    int64_t at = kept + base + before - n;
    int64_t other = p.tokens - 1 - (lo - at);  // from the end
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (lo + i < p.tokens) p.rows[mask >> i & 1 ? at++ : other--] = static_cast<int32_t>(lo + i);
    kept += all;
  }
  if (threadIdx.x == 0) {
    p.rows[p.tokens] = static_cast<int32_t>(kept);
    p.scal->kept = static_cast<int32_t>(kept);
    p.scal->hmax = p.scal->wmax = 0;
  }
}

// ---- operands ----------------------------------------------------------------------------

// The largest finite magnitude of `rows` float32 rows.
__global__ __launch_bounds__(256) void loss_most_kernel(const LossParams p, bool of_weight) {
  const int64_t rows = of_weight ? p.vocab : p.scal->kept;
  const int lane = threadIdx.x & 63;
  uint32_t most = 0;
  // A wave a row, 1024 elements on their way at a time.
  for (int64_t r = blockIdx.x * 4 + (threadIdx.x >> 6); r < rows; r += gridDim.x * 4) {
    const float* row = of_weight ? static_cast<const float*>(p.weight) + r * p.sw
                                 : static_cast<const float*>(p.hidden) + p.rows[r] * p.sh;
    for (int64_t i0 = lane * 4; i0 < p.dim; i0 += 1024) {
      float v[4][4] = {};
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (i0 + u * 256 < p.dim) ld_upto4<float>(row, i0 + u * 256, upto4(p.dim - i0 - u * 256), v[u]);
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t b = __builtin_bit_cast(uint32_t, v[u][e]) & 0x7fffffffu;
          most = b < 0x7f800000u && b > most ? b : most;
        }
    }
  }
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) {
    const uint32_t o = __shfl_xor(most, s);
    most = o > most ? o : most;
  }
  if ((threadIdx.x & 63) == 0 && most > 0) atomicMax(of_weight ? &p.scal->wmax : &p.scal->hmax, most);
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
      st4_elem<T>(static_cast<T*>(to) + at, i, v);
    }
  }
}

template <typename T> __global__ __launch_bounds__(256) void loss_gather_kernel(const LossParams p) {
  const int64_t i = (p.first + blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t kept = p.scal->kept;
  if (i >= (kept + kLossTile - 1) / kLossTile * kLossTile) return;
  const float up = pow2(up_exponent(p.scal->hmax));
  const int64_t t = i < kept ? p.rows[i] : 0;
  const T* from = i < kept ? static_cast<const T*>(p.hidden) + t * p.sh : nullptr;
  if (p.target != nullptr && (threadIdx.x & 63) == 0)
    p.target[i] = i < kept ? static_cast<int32_t>(id_at(p, t)) : -1;
  lay_row<T>(from, p.hrows, i * p.dpad, p.tpad * p.dpad, p.dim, p.dpad, up, threadIdx.x & 63);
}

template <typename T> __global__ __launch_bounds__(256) void loss_weight_kernel(const LossParams p) {
  const int64_t v = (p.first + blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (v >= p.vocab) return;
  const float up = pow2(up_exponent(p.scal->wmax));
  lay_row<T>(static_cast<const T*>(p.weight) + v * p.sw, p.wrows, v * p.dpad, p.vocab * p.dpad, p.dim, p.dpad, up,
             threadIdx.x & 63);
}

// ---- the products ---------------------------------------------------------------------------

template <typename T> using Kept = std::conditional_t<std::is_same_v<T, float>, f16, T>;
template <typename T> constexpr int kRuns = std::is_same_v<T, float> ? 3 : 1;

// What takes the scaling of float32 operands back, and log2(e) c with it.
template <typename T> __device__ __forceinline__ float logit_back(const LossParams& p) {
  if constexpr (!std::is_same_v<T, float>) return 1.f;
  return pow2(-up_exponent(p.scal->hmax)) * pow2(-up_exponent(p.scal->wmax));
}
template <typename T> __device__ __forceinline__ float logit_scale(const LossParams& p) {
  return kLog2e / p.temperature * logit_back<T>(p);
}

__device__ __forceinline__ Operand rows_operand(const LossParams& p) {
  return {p.hrows, p.dpad, p.tpad * p.dpad, p.tpad * p.dpad};
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
  if (!tile_of(blockIdx.x, (p.vocab + kLossTile - 1) / kLossTile, (kept + kLossTile - 1) / kLossTile, mt, nt)) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t v0 = mt * kLossTile + (wave >> 2) * kLossPart, t0 = nt * kLossTile + (wave & 3) * 64 + (lane & 31);
  // What the epilogue needs is on its way before the product.
  const float c = logit_scale<T>(p), back = logit_back<T>(p);
  const int32_t target[2] = {p.target != nullptr ? p.target[t0] : -1, p.target != nullptr ? p.target[t0 + 32] : -1};
  constexpr int runs = kRuns<T>;
  const ProductParams q = {weight_operand(p, 0), rows_operand(p), p.dpad, runs};
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
    const float m2 = m == -INFINITY ? 0.f : m * c, off = m == -INFINITY ? 0.f : fmaf(m, c, -m2);
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) s += fast_exp2(fmaf(acc.v[j][i][e], c, -m2));
    s += __shfl_xor(s, 32);
    s = fmaf(s, -kLn2 * off, s);
    if (lane < 32 && v0 < p.vocab) p.part[(v0 / kLossPart) * p.tpad + t] = make_float2(m * back, s);
  }
}

// The same product over a piece of the vocabulary, to ds in 16 bits.
template <typename T> __global__ __launch_bounds__(512, 2) void loss_grad_kernel(const LossParams p, int64_t vp) {
  using E = Kept<T>;
  const int64_t kept = p.scal->kept;
  int64_t mt, nt;
  if (!tile_of(blockIdx.x, p.vpiece / kLossTile, (kept + kLossTile - 1) / kLossTile, mt, nt)) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t v0 = mt * kLossTile + (wave >> 2) * 128, t0 = nt * kLossTile + (wave & 3) * 64 + (lane & 31);
  const float c = logit_scale<T>(p), up = kUp<E> / p.scal->unit;
  float a[2], b[2], m2[2];
  int32_t target[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int64_t t = t0 + j * 32;
    a[j] = p.coef[t] * up;
    b[j] = p.coef[p.tpad + t] * up;
    m2[j] = p.coef[2 * p.tpad + t];
    target[j] = p.target != nullptr ? p.target[t] : -1;
  }
  constexpr int runs = kRuns<T>;
  const ProductParams q = {weight_operand(p, vp), rows_operand(p), p.dpad, runs};
  MCPU_TILE_LDS(a0, b0, a1, b1);
  Acc acc;
  tile_product<E, false, false>(q, mt * kLossTile, nt * kLossTile, 0, static_cast<int>(p.dpad / kLossDepth) * runs,
                                a0, b0, a1, b1, acc);
  const bool edge = vp + (mt + 1) * kLossTile > p.vocab || (nt + 1) * kLossTile > kept;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int64_t t = t0 + j * 32;
    each_row(acc.v[j], [&](float x, int) { return a[j] * fast_exp2(fmaf(x, c, -m2[j])); });
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

// Distillation: the ids' places of ds, a_t exp(c s - L) less all shares of that id. A wave a row.
template <typename T> __global__ __launch_bounds__(256) void loss_place_kernel(const LossParams p, int64_t vp) {
  using E = Kept<T>;
  const int lane = threadIdx.x & 63;
  const int64_t i = (p.first + blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (i >= p.scal->kept) return;
  const int64_t t = p.rows[i];
  const int k = static_cast<int>(p.k);
  const float up = kUp<E> / p.scal->unit, c = kLog2e / p.temperature;
  const float a = p.coef[i] * up, b = p.coef[p.tpad + i] * up, m2 = p.coef[2 * p.tpad + i];
  for (int e = lane; e < k; e += 64) {
    const int64_t id = id_at(p, t * k + e);
    const int64_t v = id - vp;
    if (id < 0 || id >= p.vocab || v < 0 || v >= p.vpiece) continue;
    float q = 0.f;
    for (int o = 0; o < k; ++o) q += id_at(p, t * k + o) == id ? p.share[t * k + o] : 0.f;
    const float g = a * fast_exp2(fmaf(p.picked[t * k + e], c, -m2)) - b * q;
    uint16_t* out = static_cast<uint16_t*>(p.grad) + i * p.vpiece + v;
    *out = __builtin_bit_cast(uint16_t, from_f32<E>(g));
    if constexpr (std::is_same_v<T, float>) {
      f16 h, l;
      split_f16(g, h, l);
      out[p.tpad * p.vpiece] = __builtin_bit_cast(uint16_t, l);
    }
  }
}

// dhidden over a piece: m along the dim, n along the tokens, terms along the vocabulary.
template <typename T>
__global__ __launch_bounds__(512, 2) void loss_dhidden_kernel(const LossParams p, int64_t vp, bool add) {
  using E = Kept<T>;
  const int64_t kept = p.scal->kept;
  const int64_t mts = (p.dpad + kLossTile - 1) / kLossTile, nts = (kept + kLossTile - 1) / kLossTile;
  int64_t mt, ns;
  if (!tile_of(blockIdx.x, mts, nts * p.hsplit, mt, ns)) return;
  const int64_t nt = ns / p.hsplit;
  const int split = static_cast<int>(ns - nt * p.hsplit);
  constexpr int runs = kRuns<T>;
  const ProductParams q = {weight_operand(p, vp), grad_operand(p), p.vpiece, runs};
  const int depths = static_cast<int>(p.vpiece / kLossDepth) * runs;
  MCPU_TILE_LDS(a0, b0, a1, b1);
  Acc acc;
  tile_product<E, true, false>(q, mt * kLossTile, nt * kLossTile, static_cast<int>(int64_t{depths} * split / p.hsplit),
                               static_cast<int>(int64_t{depths} * (split + 1) / p.hsplit), a0, b0, a1, b1, acc);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int64_t t = nt * kLossTile + (wave & 3) * 64 + j * 32 + (lane & 31);
    float* out = p.acc + (split * p.tpad + t) * p.dpad;
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

// dhidden in its own type: the splits' sum; rows that do not count have none. A wave a row.
template <typename T> __global__ __launch_bounds__(256) void loss_dhidden_out_kernel(const LossParams p) {
  using E = Kept<T>;
  const int lane = threadIdx.x & 63;
  const int64_t i = (p.first + blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (i >= p.tokens) return;
  const bool in = i < p.scal->kept;
  float scale = p.scal->unit / kUp<E>;
  if constexpr (std::is_same_v<T, float>) scale *= pow2(-up_exponent(p.scal->wmax));
  T* out = static_cast<T*>(p.dhidden) + p.rows[i] * p.dim;
  for (int64_t d = lane * 4; d < p.dim; d += 256) {
    float v[4] = {};
    if (in)
      for (int s = 0; s < p.hsplit; ++s) {
        const float4 o = *reinterpret_cast<const float4*>(p.acc + (s * p.tpad + i) * p.dpad + d);
        v[0] += o.x, v[1] += o.y, v[2] += o.z, v[3] += o.w;
      }
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = in ? v[e] * scale : 0.f;
    st_upto4<T>(out, d, upto4(p.dim - d), v);
  }
}

// dweight of a piece: m along the dim, n along the vocabulary, terms along the tokens.
template <typename T>
__global__ __launch_bounds__(512, 2) void loss_dweight_kernel(const LossParams p, int64_t vp) {
  using E = Kept<T>;
  const int64_t mts = (p.dpad + kLossTile - 1) / kLossTile;
  int64_t mt, ns;
  if (!tile_of(blockIdx.x, mts, p.vpiece / kLossTile * p.wsplit, mt, ns)) return;
  const int64_t nt = ns / p.wsplit;
  const int split = static_cast<int>(ns - nt * p.wsplit);
  constexpr int runs = kRuns<T>;
  const int64_t depth = (int64_t{p.scal->kept} + kLossDepth - 1) / kLossDepth * kLossDepth;
  const ProductParams q = {rows_operand(p), grad_operand(p), depth, runs};
  const int depths = static_cast<int>(depth / kLossDepth) * runs;
  MCPU_TILE_LDS(a0, b0, a1, b1);
  Acc acc;
  tile_product<E, true, true>(q, mt * kLossTile, nt * kLossTile,
                              static_cast<int>(int64_t{depths} * split / p.wsplit),
                              static_cast<int>(int64_t{depths} * (split + 1) / p.wsplit), a0, b0, a1, b1, acc);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  float scale = p.scal->unit / kUp<E>;
  if constexpr (std::is_same_v<T, float>) scale *= pow2(-up_exponent(p.scal->hmax));
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

// dweight of a piece from its splits. A wave a row.
template <typename T> __global__ __launch_bounds__(256) void loss_dweight_out_kernel(const LossParams p, int64_t vp) {
  const int lane = threadIdx.x & 63;
  const int64_t vl = (p.first + blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (vl >= p.vpiece || vp + vl >= p.vocab) return;
  T* out = static_cast<T*>(p.dweight) + (vp + vl) * p.dim;
  for (int64_t d = lane * 4; d < p.dim; d += 256) {
    float v[4] = {};
    for (int s = 0; s < p.wsplit; ++s) {
      const float4 o = *reinterpret_cast<const float4*>(p.dwpart + (s * p.vpiece + vl) * p.dpad + d);
      v[0] += o.x, v[1] += o.y, v[2] += o.z, v[3] += o.w;
    }
    st_upto4<T>(out, d, upto4(p.dim - d), v);
  }
}

// ---- the loss of a row, and of all ------------------------------------------------------------

// 32 tokens a workgroup: eight threads a token join the parts, one takes the loss.
__global__ __launch_bounds__(256) void loss_join_kernel(const LossParams p) {
  __shared__ float ms[8][33], ss[8][33];
  const int64_t kept = p.scal->kept;
  const int64_t i = (p.first + blockIdx.x) * 32 + (threadIdx.x & 31);
  const int slice = threadIdx.x >> 5;
  const int64_t parts = (p.vocab + kLossPart - 1) / kLossPart;
  const float c = kLog2e / p.temperature;
  float m = -INFINITY, s = 0.f;
  if (i < kept) {
    for (int64_t q0 = slice; q0 < parts; q0 += 64) {
      float2 x[8];
      float top = m;
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        x[u] = q0 + u * 8 < parts ? p.part[(q0 + u * 8) * p.tpad + i] : make_float2(-INFINITY, 0.f);
        top = fmaxf(top, x[u].x);
      }
      const float sub = top == -INFINITY ? 0.f : top;
      s *= fast_exp2((m - sub) * c);
#pragma unroll
      for (int u = 0; u < 8; ++u) s = fmaf(x[u].y, fast_exp2((x[u].x - sub) * c), s);
      m = top;
    }
  }
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
  for (int q = 1; q < 8; ++q) top = fmaxf(top, ms[q][x]);
  const float sub = top == -INFINITY ? 0.f : top;
  float sum = 0.f;
  for (int q = 0; q < 8; ++q) sum = fmaf(ss[q][x], fast_exp2((ms[q][x] - sub) * c), sum);
  float* stat = p.stat + i;
  if (p.teacher == nullptr) {
    // The target joins the others: relative to their maximum, as long as that is in float32's range.
    const float own = p.picked[i], d = own - top;
    const bool far = !(d <= 40.f);
    const float mine = far ? 1.f : fast_exp2(d * c), others = far ? sum * fast_exp2(-d * c) : sum;
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

// Coefficients of the rows that count, and the unit their gradients are kept in: the
// largest coefficient itself, so that where all are alike, as under a mean, a
// target's ds of nearly -unit is not rounded the same way in every row. One workgroup.
__global__ __launch_bounds__(1024) void loss_coef_kernel(const LossParams p) {
  __shared__ float tops[16];
  const int32_t kept = p.rows[p.tokens];
  const float share = p.reduction == MCPU_REDUCE_MEAN ? 1.f / static_cast<float>(kept > 0 ? kept : 1) : 1.f;
  const float c = kLog2e / p.temperature;
  const bool each = p.reduction == MCPU_REDUCE_NONE;
  const float all = each ? 0.f : p.dloss[0] * share;
  float most = 0.f;
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
      const float m2 = stat[0][u] * c, off = fmaf(stat[0][u], c, -m2);
      p.coef[i] = a / stat[1][u] * fmaf(-kLn2, off, 1.f);
      // Cross entropy: the target's ds, a p - g = (a - g) p - g (1 - p).
      p.coef[p.tpad + i] = p.share != nullptr ? g[u] : e[u] * stat[2][u] - g[u] * stat[3][u];
      p.coef[2 * p.tpad + i] = m2;
      const float top = fmaxf(__builtin_fabsf(a), __builtin_fabsf(g[u]));
      if (top < INFINITY) most = fmaxf(most, top);
    }
  }
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) most = fmaxf(most, __shfl_xor(most, s));
  if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = most;
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int i = 1; i < 16; ++i) most = fmaxf(most, tops[i]);
  p.scal->kept = kept;
  p.scal->hmax = p.scal->wmax = 0;
  p.scal->unit = most == 0.f ? 1.f : fmaxf(most, 0x1p-100f);
}

// ---- launches -----------------------------------------------------------------------------------

template <typename K, typename... A>
void run(K kernel, LossParams p, int64_t groups, int threads, hipStream_t st, A... more) {
  launch_all(groups, threads, [&](int64_t first, unsigned count) {
    p.first = first;
    hipLaunchKernelGGL(kernel, dim3(count), dim3(threads), 0, st, p, more...);
  });
}

template <typename T> void lay_operands(const LossParams& p, hipStream_t st) {
  if constexpr (std::is_same_v<T, float>) {
    run(loss_most_kernel, p, std::min<int64_t>((p.tokens + 3) / 4, 2048), 256, st, false);
    run(loss_most_kernel, p, std::min<int64_t>((p.vocab + 3) / 4, 2048), 256, st, true);
  }
  run(loss_gather_kernel<T>, p, p.tpad / 4, 256, st);
  if (p.wrows != nullptr) run(loss_weight_kernel<T>, p, (p.vocab + 3) / 4, 256, st);
}

template <typename T> hipError_t fwd(const LossParams& p, hipStream_t st) {
  if (p.teacher != nullptr)
    run(loss_teacher_kernel<T>, p, (p.tokens + 3) / 4, 256, st);
  run(loss_rows_kernel, p, 1, 1024, st);
  lay_operands<T>(p, st);
  const int64_t vt = (p.vocab + kLossTile - 1) / kLossTile, tt = p.tpad / kLossTile;
  run(loss_logits_kernel<T>, p, vt * tt, 512, st);
  run(loss_join_kernel, p, (p.tokens + 31) / 32, 256, st);
  if (p.reduction != MCPU_REDUCE_NONE) run(loss_sum_kernel, p, 1, 1024, st);
  return hipGetLastError();
}

template <typename T> hipError_t bwd(const LossParams& p, hipStream_t st) {
  run(loss_coef_kernel, p, 1, 1024, st);
  lay_operands<T>(p, st);
  const int64_t tt = p.tpad / kLossTile, vt = p.vpiece / kLossTile, dt = (p.dpad + kLossTile - 1) / kLossTile;
  for (int64_t vp = 0; vp < p.vocab; vp += p.vpiece) {
    run(loss_grad_kernel<T>, p, vt * tt, 512, st, vp);
    if (p.share != nullptr) run(loss_place_kernel<T>, p, (p.tokens + 3) / 4, 256, st, vp);
    if (p.dhidden != nullptr) run(loss_dhidden_kernel<T>, p, dt * tt * p.hsplit, 512, st, vp, vp > 0);
    if (p.dweight != nullptr) {
      run(loss_dweight_kernel<T>, p, dt * vt * p.wsplit, 512, st, vp);
      if (p.dwpart != nullptr) run(loss_dweight_out_kernel<T>, p, vt * kLossTile / 4, 256, st, vp);
    }
  }
  if (p.dhidden != nullptr) run(loss_dhidden_out_kernel<T>, p, (p.tokens + 3) / 4, 256, st);
  return hipGetLastError();
}

}  // namespace

// Splits of a product's terms, for `tiles` results of 256 KiB over `depths` each: what 256 workgroups at a
// time take, at 4.6 TFLOP/s each, and 4 TB/s for the splits' results, written and read.
static int splits_for(int64_t tiles, int64_t depths) {
  int best = 1;
  double least = 0;
  for (int s = 1; s <= 64 && (s == 1 || depths / s >= 8); ++s) {
    const double rounds = static_cast<double>((tiles * s + 255) / 256), each = static_cast<double>(depths) / s;
    const double us = rounds * (each * 1.8 + 6) + (s > 1 ? tiles * s * 0.131 : 0);
    if (s == 1 || us < 0.97 * least) best = s, least = us;
  }
  return best;
}

void loss_plan(LossParams& p) {
  const int pieces = loss_pieces(p.dtype);
  auto up = [](int64_t n, int64_t to) { return (n + to - 1) / to * to; };
  p.tpad = up(p.tokens, kLossTile);
  p.dpad = up(p.dim, kLossDepth);
  const int64_t most = std::max<int64_t>(1, (int64_t{1} << 29) / pieces / p.tpad / kLossTile) * kLossTile;
  const int64_t count = (p.vocab + most - 1) / most;
  p.vpiece = up((p.vocab + count - 1) / count, kLossTile);
  const int64_t dt = (p.dpad + kLossTile - 1) / kLossTile;
  p.hsplit = splits_for(dt * (p.tpad / kLossTile), p.vpiece / kLossDepth * (pieces == 2 ? 3 : 1));
  p.wsplit = splits_for(dt * (p.vpiece / kLossTile), p.tpad / kLossDepth * (pieces == 2 ? 3 : 1));
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
