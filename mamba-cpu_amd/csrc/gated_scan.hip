// Gated linear recurrence on gfx950: forward, backward and the single-token
// step. Per batch row, step t and channel d, all in float32:
//
//   rho = sigmoid(a_gate)   iota = sigmoid(x_gate)   s = c softplus(decay_d) rho
//   a = exp(-s)             m = sqrt(1 - exp(-2 s))
//   h_t = k_t a h_{t-1} + m iota x_t,   y_t = h_t
//
// with k_t = 0 at the first step of another sequence of a packed row, else 1.
// The step h -> a h + b composes as (P, S): h -> P h + S, so time is split: a
// wave takes kGatedT consecutive steps of 64 channels in its registers, forms
// their (P, S), the workgroup's waves exchange theirs through LDS, and each
// wave then knows the state in front of its segment. A wave's lanes are 64
// neighbouring channels, so each of its loads is a run of one row.
//
// Backward, with g_t = dL/dh_t:  g_t = dy_t + k_{t+1} a_{t+1} g_{t+1},
//   dx = g m iota          dx_gate = dx x (1 - iota)
//   e  = g (iota x a^2 / m - k a h_{t-1})
//   da_gate = e s (1 - rho)       ddecay = sum e c rho sigmoid(decay)
// is the same scan from the other end; the states it needs are recomputed
// from the one the forward kept in front of every segment, in float32 (the
// stored y may be 16 bits wide).
#include "gated_scan.h"
#include "lm_math.h"

namespace mcpu {
namespace {

// 1 - exp(-y) for y >= 0, given ey = exp(-y): below 1/2 its series, whose
// first dropped term is y^9 / 9!, above it the difference, which loses less than two bits.
__device__ __forceinline__ float one_minus_exp(float y, float ey) {
  float q = -1.f / 40320.f;
  q = fmaf(q, y, 1.f / 5040.f);
  q = fmaf(q, y, -1.f / 720.f);
  q = fmaf(q, y, 1.f / 120.f);
  q = fmaf(q, y, -1.f / 24.f);
  q = fmaf(q, y, 1.f / 6.f);
  q = fmaf(q, y, -0.5f);
  q = fmaf(q, y, 1.f);
  return y < 0.5f ? y * q : 1.0f - ey;
}

struct Gates {
  float rho, nrho, iota, niota, s, a, m;
};
__device__ __forceinline__ Gates gates(float a_gate, float x_gate, float csp) {
  Gates g;
  g.rho = sigmoid_acc(a_gate, g.nrho);
  g.iota = sigmoid_acc(x_gate, g.niota);
  g.s = csp * g.rho;
  g.a = exp_acc(-g.s);
  g.m = __builtin_amdgcn_sqrtf(one_minus_exp(2.0f * g.s, g.a * g.a));
  return g;
}

// Whether step t starts another sequence than step t - 1 of its row.
__device__ __forceinline__ bool starts(const int32_t* ids, int64_t t) {
  return ids != nullptr && t > 0 && ids[t] != ids[t - 1];
}

template <typename T>
__global__ __launch_bounds__(64 * kGatedWaves) void gated_fwd_kernel(const GatedScanParams p) {
  constexpr int TS = kGatedT, W = kGatedWaves;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t tiles = (p.dim + 63) / 64;
  const int64_t b = blockIdx.x / tiles, d = (blockIdx.x % tiles) * 64 + lane;
  const bool live = d < p.dim;
  const int64_t dd = live ? d : 0;
  const T* x = static_cast<const T*>(p.x) + b * p.sx[0] + dd * p.sx[2];
  const T* ag = static_cast<const T*>(p.a_gate) + b * p.sa[0] + dd * p.sa[2];
  const T* ig = static_cast<const T*>(p.x_gate) + b * p.si[0] + dd * p.si[2];
  T* y = static_cast<T*>(p.y) + b * p.sy[0] + dd * p.sy[2];
  const int32_t* ids = p.seq_idx == nullptr ? nullptr : p.seq_idx + b * p.len;
  const int64_t nseg = (p.len + TS - 1) / TS;
  const float csp = p.c * softplus_acc(p.decay[dd]);
  float carry = p.init == nullptr ? 0.f : p.init[b * p.dim + dd];
  __shared__ float aggP[2][W][64], aggS[2][W][64];
  int buf = 0;
  for (int64_t t0 = 0; t0 < p.len; t0 += W * TS, buf ^= 1) {
    const int64_t ts = t0 + w * TS;
    float a[TS], u[TS], P = 1.f, S = 0.f;
#pragma unroll
    for (int i = 0; i < TS; ++i) {
      const int64_t t = ts + i;
      a[i] = 1.f;
      u[i] = 0.f;
      if (t < p.len) {
        const Gates g = gates(to_f32(ag[t * p.sa[1]]), to_f32(ig[t * p.si[1]]), csp);
        a[i] = starts(ids, t) ? 0.f : g.a;
        u[i] = g.m * g.iota * to_f32(x[t * p.sx[1]]);
      }
      S = fmaf(a[i], S, u[i]);
      P *= a[i];
    }
    aggP[buf][w][lane] = P;
    aggS[buf][w][lane] = S;
    __syncthreads();
    float h = carry;
    for (int v = 0; v < W; ++v) {
      if (v == w) h = carry;
      carry = fmaf(aggP[buf][v][lane], carry, aggS[buf][v][lane]);
    }
    if (live && ts < p.len) {
      if (p.ckpt != nullptr) p.ckpt[(b * nseg + ts / TS) * p.dim + d] = h;
#pragma unroll
      for (int i = 0; i < TS; ++i) {
        h = fmaf(a[i], h, u[i]);
        if (ts + i < p.len) y[(ts + i) * p.sy[1]] = from_f32<T>(h);
      }
    }
  }
  if (live && w == 0 && p.last != nullptr) p.last[b * p.dim + d] = carry;
}

template <typename T>
__global__ __launch_bounds__(64 * kGatedWaves) void gated_bwd_kernel(const GatedScanParams p) {
  constexpr int TS = kGatedT, W = kGatedWaves;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t tiles = (p.dim + 63) / 64;
  const int64_t b = blockIdx.x / tiles, d = (blockIdx.x % tiles) * 64 + lane;
  const bool live = d < p.dim;
  const int64_t dd = live ? d : 0;
  const T* x = static_cast<const T*>(p.x) + b * p.sx[0] + dd * p.sx[2];
  const T* ag = static_cast<const T*>(p.a_gate) + b * p.sa[0] + dd * p.sa[2];
  const T* ig = static_cast<const T*>(p.x_gate) + b * p.si[0] + dd * p.si[2];
  const T* dy = static_cast<const T*>(p.dy) + b * p.sdy[0] + dd * p.sdy[2];
  T* dx = static_cast<T*>(p.dx) + b * p.sdx[0] + dd * p.sdx[2];
  T* dag = static_cast<T*>(p.da_gate) + b * p.sda[0] + dd * p.sda[2];
  T* dig = static_cast<T*>(p.dx_gate) + b * p.sdi[0] + dd * p.sdi[2];
  const int32_t* ids = p.seq_idx == nullptr ? nullptr : p.seq_idx + b * p.len;
  const int64_t nseg = (p.len + TS - 1) / TS;
  const float lam = p.decay[dd];
  const float csp = p.c * softplus_acc(lam);
  float carry = p.dlast == nullptr ? 0.f : p.dlast[b * p.dim + dd];
  float acc = 0.f;  // sum over this lane's steps of e rho
  __shared__ float aggP[2][W][64], aggS[2][W][64];
  int buf = 0;
  const int64_t nchunk = (p.len + W * TS - 1) / (W * TS);
  for (int64_t ch = nchunk - 1; ch >= 0; --ch, buf ^= 1) {
    const int64_t ts = ch * (W * TS) + w * TS;
    float ka[TS], hp[TS];
    float h = ts < p.len ? p.ckpt[(b * nseg + ts / TS) * p.dim + dd] : 0.f;
    float P = 1.f, S = 0.f;
#pragma unroll
    for (int i = 0; i < TS; ++i) {
      const int64_t t = ts + i;
      ka[i] = 1.f;
      hp[i] = h;
      if (t < p.len) {
        const Gates g = gates(to_f32(ag[t * p.sa[1]]), to_f32(ig[t * p.si[1]]), csp);
        ka[i] = starts(ids, t) ? 0.f : g.a;
        h = fmaf(ka[i], h, g.m * g.iota * to_f32(x[t * p.sx[1]]));
      }
      P *= ka[i];
    }
#pragma unroll
    for (int i = TS - 1; i >= 0; --i) {
      const int64_t t = ts + i;
      S = ka[i] * (S + (t < p.len ? to_f32(dy[t * p.sdy[1]]) : 0.f));
    }
    aggP[buf][w][lane] = P;
    aggS[buf][w][lane] = S;
    __syncthreads();
    float G = carry;
    for (int v = W - 1; v >= 0; --v) {
      if (v == w) G = carry;
      carry = fmaf(aggP[buf][v][lane], carry, aggS[buf][v][lane]);
    }
#pragma unroll
    for (int i = TS - 1; i >= 0; --i) {
      const int64_t t = ts + i;
      if (t < p.len) {
        const float xv = to_f32(x[t * p.sx[1]]);
        const Gates q = gates(to_f32(ag[t * p.sa[1]]), to_f32(ig[t * p.si[1]]), csp);
        const float g = to_f32(dy[t * p.sdy[1]]) + G;
        const float dxv = g * q.m * q.iota;
        // m = 0 (a closed gate, s underflown): the limit of a^2 s / m is 0.
        const float inv = q.m > 0.f ? fast_rcp(q.m) : 0.f;
        const float e = g * (q.iota * xv * (q.a * q.a * inv) - ka[i] * hp[i]);
        if (live) {
          dx[t * p.sdx[1]] = from_f32<T>(dxv);
          dig[t * p.sdi[1]] = from_f32<T>(dxv * xv * q.niota);
          dag[t * p.sda[1]] = from_f32<T>(e * q.s * q.nrho);
        }
        acc = fmaf(e, q.rho, acc);
        G = ka[i] * g;
      }
    }
  }
  if (live && w == 0 && p.dinit != nullptr) p.dinit[b * p.dim + d] = carry;
  __syncthreads();
  aggP[0][w][lane] = acc;
  __syncthreads();
  if (w == 0 && live) {
    float sum = 0.f;
    for (int v = 0; v < W; ++v) sum += aggP[0][v][lane];
    float n;
    p.ddecay_part[b * p.dim + d] = sum * p.c * sigmoid_acc(lam, n);
  }
}

// ddecay: the partial sums of the batch rows, added in order.
__global__ __launch_bounds__(256) void gated_ddecay_kernel(const GatedScanParams p) {
  const int64_t d = blockIdx.x * 256ll + threadIdx.x;
  if (d >= p.dim) return;
  float sum = 0.f;
  for (int64_t b = 0; b < p.batch; ++b) sum += p.ddecay_part[b * p.dim + d];
  p.ddecay[d] = sum;
}

// One token: state (rows, dim) float32 in place.
template <typename T>
__global__ __launch_bounds__(256) void gated_step_kernel(const GatedStepParams p) {
  const int64_t n = blockIdx.x * 256ll + threadIdx.x;
  if (n >= p.batch * p.dim) return;
  const int64_t b = n / p.dim, d = n % p.dim;
  const int64_t row = p.state_idx == nullptr ? b : p.state_idx[b];
  T* y = static_cast<T*>(p.y) + n;
  if (row < 0 || row >= p.state_batch) {
    *y = from_f32<T>(0.f);
    return;
  }
  const Gates g = gates(ld<T>(p.a_gate, b * p.sa[0] + d * p.sa[1]), ld<T>(p.x_gate, b * p.si[0] + d * p.si[1]),
                        p.c * softplus_acc(p.decay[d]));
  float* h = p.state + row * p.sst[0] + d * p.sst[1];
  const float v = fmaf(g.a, *h, g.m * g.iota * ld<T>(p.x, b * p.sx[0] + d * p.sx[1]));
  *h = v;
  *y = from_f32<T>(v);
}

template <typename F> hipError_t by_dtype(int dtype, F&& f) {
  if (dtype == MCPU_F32) f(float{});
  else if (dtype == MCPU_BF16) f(bf16{});
  else f(f16{});
  return hipGetLastError();
}

}  // namespace

hipError_t gated_scan_fwd_launch(const GatedScanParams& p, int dtype, hipStream_t st) {
  const unsigned grid = static_cast<unsigned>((p.dim + 63) / 64 * p.batch);
  return by_dtype(dtype, [&](auto t) {
    hipLaunchKernelGGL(gated_fwd_kernel<decltype(t)>, dim3(grid), dim3(64 * kGatedWaves), 0, st, p);
  });
}

hipError_t gated_scan_bwd_launch(const GatedScanParams& p, int dtype, hipStream_t st) {
  const unsigned grid = static_cast<unsigned>((p.dim + 63) / 64 * p.batch);
  const hipError_t e = by_dtype(dtype, [&](auto t) {
    hipLaunchKernelGGL(gated_bwd_kernel<decltype(t)>, dim3(grid), dim3(64 * kGatedWaves), 0, st, p);
  });
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(gated_ddecay_kernel, dim3(static_cast<unsigned>((p.dim + 255) / 256)), dim3(256), 0, st, p);
  return hipGetLastError();
}

hipError_t gated_step_launch(const GatedStepParams& p, int dtype, hipStream_t st) {
  const unsigned grid = static_cast<unsigned>((p.batch * p.dim + 255) / 256);
  return by_dtype(dtype, [&](auto t) {
    hipLaunchKernelGGL(gated_step_kernel<decltype(t)>, dim3(grid), dim3(256), 0, st, p);
  });
}

}  // namespace mcpu
