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
// these. The few products with the ids' rows are formed by themselves.
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

// ---- labels: the ids' products, the teacher's distribution, which rows count ---------------

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

// Cross entropy: 16 lanes a token.
template <typename T> __global__ __launch_bounds__(256) void loss_target_kernel(const LossParams p) {
  const int64_t t = (p.first + blockIdx.x) * 16 + (threadIdx.x >> 4);
  if (t >= p.tokens) return;
  const int j = threadIdx.x & 15;
  const int64_t id = id_at(p, t);
  const bool keep = id >= 0 && id < p.vocab && id != p.ignore;
  float s = 0.f;
  if (keep)
    s = dot16<T>(static_cast<const T*>(p.hidden) + t * p.sh, static_cast<const T*>(p.weight) + id * p.sw, p.dim, j);
  if (j == 0) {
    p.keep[t] = keep;
    p.picked[t] = s;
  }
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
  float neg = 0.f;
  for (int i = lane; i < k; i += 64) {
    float q = 0.f;
    if (in(i) && !(teacher[i] == -INFINITY)) {
      const float x = (teacher[i] - m) * c;
      q = exp_acc(x) * inv;
      if (!(q == 0.f)) neg = fmaf(q, x - logsum, neg);
    }
    share[i] = q;
  }
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) neg += __shfl_xor(neg, s);
  if (lane == 0) {
    p.keep[t] = keep;
    p.neg[t] = neg;
  }
  const int j = lane & 15;
  for (int i = lane >> 4; i < k; i += 4) {
    const int64_t id = id_at(p, t * k + i);
    float s = 0.f;
    if (keep && id >= 0 && id < p.vocab)
      s = dot16<T>(static_cast<const T*>(p.hidden) + t * p.sh, static_cast<const T*>(p.weight) + id * p.sw, p.dim, j);
    if (j == 0) p.picked[t * k + i] = s;
  }
}

// The rows that count, in order, then the others; one workgroup.
__global__ __launch_bounds__(1024) void loss_rows_kernel(const LossParams p) {
  __shared__ int32_t sums[16];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int64_t per = (p.tokens + 1023) / 1024;
  const int64_t lo = threadIdx.x * per < p.tokens ? threadIdx.x * per : p.tokens;
  const int64_t hi = lo + per < p.tokens ? lo + per : p.tokens;
  int32_t n = 0;
  for (int64_t t = lo; t < hi; ++t) n += p.keep[t];
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
  int64_t kept = base + before - n;
  int64_t other = all + (lo - kept);
  for (int64_t t = lo; t < hi; ++t) p.rows[p.keep[t] ? kept++ : other++] = static_cast<int32_t>(t);
  if (threadIdx.x == 0) {
    p.rows[p.tokens] = all;
    p.scal->kept = all;
    p.scal->hmax = p.scal->wmax = 0;
  }
}

// ---- operands ----------------------------------------------------------------------------

// The largest finite magnitude of `rows` float32 rows.
__global__ __launch_bounds__(256) void loss_most_kernel(const LossParams p, bool of_weight) {
  const int64_t rows = of_weight ? p.vocab : p.scal->kept;
  uint32_t most = 0;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const float* row = of_weight ? static_cast<const float*>(p.weight) + r * p.sw
                                 : static_cast<const float*>(p.hidden) + p.rows[r] * p.sh;
    for (int64_t i = threadIdx.x * 4; i < p.dim; i += 1024) {
      float v[4];
      ld_upto4<float>(row, i, upto4(p.dim - i), v);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t b = __builtin_bit_cast(uint32_t, v[e]) & 0x7fffffffu;
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
  const T* from = i < kept ? static_cast<const T*>(p.hidden) + p.rows[i] * p.sh : nullptr;
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

// log2(e) c, and what takes the scaling of float32 operands back.
__device__ __forceinline__ float logit_scale(const LossParams& p) {
  const float c = kLog2e / p.temperature;
  if (p.dtype != MCPU_F32) return c;
  return c * pow2(-up_exponent(p.scal->hmax)) * pow2(-up_exponent(p.scal->wmax));
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

// Logits of a tile of 256 vocabulary rows (m) and 256 tokens (n): per token the
// maximum and the sum of each 128 rows, in base 2.
template <typename E> __global__ __launch_bounds__(512, 2) void loss_logits_kernel(const LossParams p) {
  const int64_t kept = p.scal->kept;
  int64_t mt, nt;
  if (!tile_of(blockIdx.x, (p.vocab + kLossTile - 1) / kLossTile, (kept + kLossTile - 1) / kLossTile, mt, nt)) return;
  const int runs = p.dtype == MCPU_F32 ? 3 : 1;
  const ProductParams q = {weight_operand(p, 0), rows_operand(p), p.dpad, runs};
  Acc acc;
  tile_product<E, false, false>(q, mt * kLossTile, nt * kLossTile, 0, static_cast<int>(p.dpad / kLossDepth) * runs,
                                acc);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t v0 = mt * kLossTile + (wave >> 2) * kLossPart;
  const float c = logit_scale(p);
  if (v0 + kLossPart > p.vocab) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (v0 + 32 * i + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3) >= p.vocab)
          acc.v[i][0][e] = acc.v[i][1][e] = -INFINITY;
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) m = fmaxf(m, acc.v[i][j][e]);
    m = fmaxf(m, __shfl_xor(m, 32));
    const float m2 = m * c, sub = m == -INFINITY ? 0.f : m2;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) s += fast_exp2(fmaf(acc.v[i][j][e], c, -sub));
    s += __shfl_xor(s, 32);
    const int64_t t = nt * kLossTile + (wave & 3) * 64 + j * 32 + (lane & 31);
    if (lane < 32 && v0 < p.vocab) p.part[(v0 / kLossPart) * p.tpad + t] = make_float2(m2, s);
  }
}

// The same product over a piece of the vocabulary, to ds in 16 bits.
template <typename E> __global__ __launch_bounds__(512, 2) void loss_grad_kernel(const LossParams p, int64_t vp) {
  const int64_t kept = p.scal->kept;
  int64_t mt, nt;
  if (!tile_of(blockIdx.x, p.vpiece / kLossTile, (kept + kLossTile - 1) / kLossTile, mt, nt)) return;
  const int runs = p.dtype == MCPU_F32 ? 3 : 1;
  const ProductParams q = {weight_operand(p, vp), rows_operand(p), p.dpad, runs};
  Acc acc;
  tile_product<E, false, false>(q, mt * kLossTile, nt * kLossTile, 0, static_cast<int>(p.dpad / kLossDepth) * runs,
                                acc);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t v0 = mt * kLossTile + (wave >> 2) * 128;
  const float c = logit_scale(p), up = kUp<E> / p.scal->unit;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int64_t t = nt * kLossTile + (wave & 3) * 64 + j * 32 + (lane & 31);
    const bool in = t < kept;
    const float a = in ? p.coef[t] * up : 0.f, l2 = in ? p.coef[2 * p.tpad + t] : 0.f;
    uint16_t* out = static_cast<uint16_t*>(p.grad) + t * p.vpiece + v0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float v[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        v[e] = a * fast_exp2(fmaf(acc.v[i][j][e], c, -l2));
        if (!in || vp + v0 + 32 * i + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3) >= p.vocab) v[e] = 0.f;
      }
      // Four rows a lane become eight: the two halves of the wave trade the second of two groups of eight.
#pragma unroll
      for (int g = 0; g < 4; g += 2) {
        auto put = [&](const float* x, const float* y, uint16_t* to) {
          uint32_t x0, x1, y0, y1;
          narrow4<E>(x, x0, x1);
          narrow4<E>(y, y0, y1);
          const auto s0 = __builtin_amdgcn_permlane32_swap(x0, y0, false, false);
          const auto s1 = __builtin_amdgcn_permlane32_swap(x1, y1, false, false);
          const uint32_t r0 = s0[0], r1 = s1[0], r2 = s0[1], r3 = s1[1];
          *reinterpret_cast<u32x4*>(to + 32 * i + 8 * g + 8 * (lane >> 5)) = u32x4{r0, r1, r2, r3};
        };
        put(v + 4 * g, v + 4 * g + 4, out);
        if (p.dtype == MCPU_F32) {
          float lo[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            f16 h, l;
            split_f16(v[4 * g + e], h, l);
            lo[e] = static_cast<float>(l);
          }
          put(lo, lo + 4, out + p.tpad * p.vpiece);
        }
      }
    }
  }
}

// The ids' places of ds: a_t exp(c s - L) less all shares of that id. A wave a row.
template <typename E> __global__ __launch_bounds__(256) void loss_place_kernel(const LossParams p, int64_t vp) {
  const int lane = threadIdx.x & 63;
  const int64_t i = (p.first + blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (i >= p.scal->kept) return;
  const int64_t t = p.rows[i];
  const int k = static_cast<int>(p.k);
  const float up = kUp<E> / p.scal->unit, c = kLog2e / p.temperature;
  const float a = p.coef[i] * up, b = p.coef[p.tpad + i] * up, l2 = p.coef[2 * p.tpad + i];
  for (int e = lane; e < k; e += 64) {
    const int64_t id = id_at(p, t * k + e);
    const int64_t v = id - vp;
    if (id < 0 || id >= p.vocab || v < 0 || v >= p.vpiece) continue;
    float q = 1.f;
    if (p.share != nullptr) {
      q = 0.f;
      for (int o = 0; o < k; ++o) q += id_at(p, t * k + o) == id ? p.share[t * k + o] : 0.f;
    }
    const float g = a * fast_exp2(fmaf(p.picked[t * k + e], c, -l2)) - b * q;
    uint16_t* out = static_cast<uint16_t*>(p.grad) + i * p.vpiece + v;
    *out = __builtin_bit_cast(uint16_t, from_f32<E>(g));
    if (p.dtype == MCPU_F32) {
      f16 h, l;
      split_f16(g, h, l);
      out[p.tpad * p.vpiece] = __builtin_bit_cast(uint16_t, l);
    }
  }
}

// dhidden over a piece: m along the dim, n along the tokens, terms along the vocabulary.
template <typename E>
__global__ __launch_bounds__(512, 2) void loss_dhidden_kernel(const LossParams p, int64_t vp, bool add) {
  const int64_t kept = p.scal->kept;
  const int64_t mts = (p.dpad + kLossTile - 1) / kLossTile, nts = (kept + kLossTile - 1) / kLossTile;
  int64_t mt, ns;
  if (!tile_of(blockIdx.x, mts, nts * p.hsplit, mt, ns)) return;
  const int64_t nt = ns / p.hsplit;
  const int split = static_cast<int>(ns - nt * p.hsplit);
  const int runs = p.dtype == MCPU_F32 ? 3 : 1;
  const ProductParams q = {weight_operand(p, vp), grad_operand(p), p.vpiece, runs};
  const int depths = static_cast<int>(p.vpiece / kLossDepth) * runs;
  Acc acc;
  tile_product<E, true, false>(q, mt * kLossTile, nt * kLossTile, depths * split / p.hsplit,
                               depths * (split + 1) / p.hsplit, acc);
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
        float4 v = make_float4(acc.v[i][j][4 * g], acc.v[i][j][4 * g + 1], acc.v[i][j][4 * g + 2],
                               acc.v[i][j][4 * g + 3]);
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
template <typename T, typename E> __global__ __launch_bounds__(256) void loss_dhidden_out_kernel(const LossParams p) {
  const int lane = threadIdx.x & 63;
  const int64_t i = (p.first + blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (i >= p.tokens) return;
  const bool in = i < p.scal->kept;
  float scale = p.scal->unit / kUp<E>;
  if (p.dtype == MCPU_F32) scale *= pow2(-up_exponent(p.scal->wmax));
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
template <typename T, typename E>
__global__ __launch_bounds__(512, 2) void loss_dweight_kernel(const LossParams p, int64_t vp) {
  const int64_t mts = (p.dpad + kLossTile - 1) / kLossTile;
  int64_t mt, ns;
  if (!tile_of(blockIdx.x, mts, p.vpiece / kLossTile * p.wsplit, mt, ns)) return;
  const int64_t nt = ns / p.wsplit;
  const int split = static_cast<int>(ns - nt * p.wsplit);
  const int runs = p.dtype == MCPU_F32 ? 3 : 1;
  const int64_t depth = (int64_t{p.scal->kept} + kLossDepth - 1) / kLossDepth * kLossDepth;
  const ProductParams q = {rows_operand(p), grad_operand(p), depth, runs};
  const int depths = static_cast<int>(depth / kLossDepth) * runs;
  Acc acc;
  tile_product<E, true, true>(q, mt * kLossTile, nt * kLossTile,
                              static_cast<int>(int64_t{depths} * split / p.wsplit),
                              static_cast<int>(int64_t{depths} * (split + 1) / p.wsplit), acc);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  float scale = p.scal->unit / kUp<E>;
  if (p.dtype == MCPU_F32) scale *= pow2(-up_exponent(p.scal->hmax));
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
        for (int e = 0; e < 4; ++e) x[e] = acc.v[i][j][4 * g + e] * scale;
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
  float m = -INFINITY, s = 0.f;
  if (i < kept) {
    for (int64_t q = slice; q < parts; q += 8) {
      const float2 x = p.part[q * p.tpad + i];
      const float top = fmaxf(m, x.x), sub = top == -INFINITY ? 0.f : top;
      s = s * fast_exp2(m - sub) + x.y * fast_exp2(x.x - sub);
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
  for (int q = 0; q < 8; ++q) sum = fmaf(ss[q][x], fast_exp2(ms[q][x] - sub), sum);
  // log2 of the sum apart from the maximum, both to natural logarithms.
  const float lse = fmaf(top, kLn2, __builtin_amdgcn_logf(sum) * kLn2);
  p.lse[t] = lse;
  if (p.teacher == nullptr) {
    p.each[t] = lse - p.picked[t];
  } else {
    const float c = 1.f / p.temperature;
    float cross = 0.f;
    for (int64_t e = t * p.k; e < (t + 1) * p.k; ++e)
      if (!(p.share[e] == 0.f)) cross = fmaf(p.share[e], lse - p.picked[e] * c, cross);
    p.each[t] = (p.neg[t] + cross) * p.temperature * p.temperature;
  }
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

// Coefficients of the rows that count, and the unit their gradients are kept in; one workgroup.
__global__ __launch_bounds__(1024) void loss_coef_kernel(const LossParams p) {
  __shared__ float tops[16];
  const int32_t kept = p.rows[p.tokens];
  const float share = p.reduction == MCPU_REDUCE_MEAN ? 1.f / static_cast<float>(kept > 0 ? kept : 1) : 1.f;
  float most = 0.f;
  for (int64_t i = threadIdx.x; i < kept; i += 1024) {
    const int64_t t = p.rows[i];
    float g = p.reduction == MCPU_REDUCE_NONE ? (p.dloss != nullptr ? p.dloss[t] : 0.f) : p.dloss[0] * share;
    g *= p.teacher != nullptr || p.share != nullptr ? p.temperature : 1.f;
    const float a = p.dlse != nullptr ? g + p.dlse[t] : g;
    p.coef[i] = a;
    p.coef[p.tpad + i] = g;
    p.coef[2 * p.tpad + i] = p.lse[t] * kLog2e;
    const float top = fmaxf(__builtin_fabsf(a), __builtin_fabsf(g));
    if (top < INFINITY) most = fmaxf(most, top);
  }
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) most = fmaxf(most, __shfl_xor(most, s));
  if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = most;
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int i = 1; i < 16; ++i) most = fmaxf(most, tops[i]);
  int e = static_cast<int>(__builtin_bit_cast(uint32_t, most) >> 23) - 126;  // most < 2^e
  e = most == 0.f ? 0 : e < -100 ? -100 : e > 100 ? 100 : e;
  p.scal->kept = kept;
  p.scal->hmax = p.scal->wmax = 0;
  p.scal->unit = pow2(e);
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
    run(loss_most_kernel, p, std::min<int64_t>(p.tokens, 1024), 256, st, false);
    run(loss_most_kernel, p, std::min<int64_t>(p.vocab, 2048), 256, st, true);
  }
  run(loss_gather_kernel<T>, p, p.tpad / 4, 256, st);
  if (p.wrows != nullptr) run(loss_weight_kernel<T>, p, (p.vocab + 3) / 4, 256, st);
}

template <typename T> using Kept = std::conditional_t<std::is_same_v<T, float>, f16, T>;

template <typename T> hipError_t fwd(const LossParams& p, hipStream_t st) {
  if (p.teacher == nullptr)
    run(loss_target_kernel<T>, p, (p.tokens + 15) / 16, 256, st);
  else
    run(loss_teacher_kernel<T>, p, (p.tokens + 3) / 4, 256, st);
  run(loss_rows_kernel, p, 1, 1024, st);
  lay_operands<T>(p, st);
  const int64_t vt = (p.vocab + kLossTile - 1) / kLossTile, tt = p.tpad / kLossTile;
  run(loss_logits_kernel<Kept<T>>, p, vt * tt, 512, st);
  run(loss_join_kernel, p, (p.tokens + 31) / 32, 256, st);
  if (p.reduction != MCPU_REDUCE_NONE) run(loss_sum_kernel, p, 1, 1024, st);
  return hipGetLastError();
}

template <typename T> hipError_t bwd(const LossParams& p, hipStream_t st) {
  using E = Kept<T>;
  run(loss_coef_kernel, p, 1, 1024, st);
  lay_operands<T>(p, st);
  const int64_t tt = p.tpad / kLossTile, vt = p.vpiece / kLossTile, dt = (p.dpad + kLossTile - 1) / kLossTile;
  for (int64_t vp = 0; vp < p.vocab; vp += p.vpiece) {
    run(loss_grad_kernel<E>, p, vt * tt, 512, st, vp);
    run(loss_place_kernel<E>, p, (p.tokens + 3) / 4, 256, st, vp);
    if (p.dhidden != nullptr) run(loss_dhidden_kernel<E>, p, dt * tt * p.hsplit, 512, st, vp, vp > 0);
    if (p.dweight != nullptr) {
      run(loss_dweight_kernel<T, E>, p, dt * vt * p.wsplit, 512, st, vp);
      if (p.dwpart != nullptr) run(loss_dweight_out_kernel<T>, p, vt * kLossTile / 4, 256, st, vp);
    }
  }
  if (p.dhidden != nullptr) run(loss_dhidden_out_kernel<T, E>, p, (p.tokens + 3) / 4, 256, st);
  return hipGetLastError();
}

}  // namespace

// Splits of a product's terms that fill the GPU's workgroups best: `tiles` of `depths` each, less what a
// split's own partial result costs.
static int splits_for(int64_t tiles, int64_t depths) {
  int best = 1;
  double least = 0;
  for (int s = 1; s <= 8 && (s == 1 || depths / s >= 8); ++s) {
    const double cost = static_cast<double>((tiles * s + 255) / 256) / s * (1 + 0.02 * (s - 1));
    if (s == 1 || cost < 0.95 * least) best = s, least = cost;
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
  p.hsplit = splits_for(dt * (p.tpad / kLossTile), p.vpiece / kLossDepth);
  p.wsplit = splits_for(dt * (p.vpiece / kLossTile), p.tpad / kLossDepth);
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
