// Gated linear recurrence on gfx950: forward, backward and the single-token
// step. Per batch row, step t and channel d, all in float32:
//
//   rho = sigmoid(a_gate)   iota = sigmoid(x_gate)   s = c softplus(decay_d) rho
//   a = exp(-s)             m = sqrt(q), q = 1 - exp(-2 s)
//   h_t = k_t a h_{t-1} + m iota x_t,   y_t = h_t
//
// with k_t = 0 at the first step of another sequence of a packed row, else 1.
// The step h -> a h + b composes as (P, S): h -> P h + S, so time is split: a
// wave takes kGatedT consecutive steps of its channels in registers and forms
// their (P, S), the workgroup's waves exchange theirs through LDS, and each
// wave then knows the state in front of its segment. A lane holds `vec`
// neighbouring channels (4 bytes where the operands allow), so that a wave
// reads 256 bytes of a row at once.
//
// Where the channels alone do not fill the chip, a row's steps are split over
// workgroups too: a first launch forms the (P, S) of every split but the last,
// the second starts each split from the composition of those before it. It
// reads the inputs twice; a single launch of few workgroups is slower (the
// rule and both sides: gated_scan_plan).
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

constexpr int TS = kGatedT, W = kGatedWaves;

// ---- VC neighbouring channels of a row -------------------------------------------------

template <int BYTES> struct WordOf;
template <> struct WordOf<2> { using type = uint16_t; };
template <> struct WordOf<4> { using type = uint32_t; };
template <> struct WordOf<8> { using type = uint2; };
template <typename T, int VC> using Word = typename WordOf<sizeof(T) * VC>::type;

template <typename T, int VC> __device__ __forceinline__ void widen(Word<T, VC> r, float (&v)[VC]) {
  if constexpr (sizeof(T) == 4 && VC == 1) {
    v[0] = __builtin_bit_cast(float, r);
  } else if constexpr (VC == 1) {
    v[0] = to_f32(__builtin_bit_cast(T, r));
  } else {
    static_assert(sizeof(T) == 2 && VC == 2);
    v[0] = to_f32(__builtin_bit_cast(T, static_cast<uint16_t>(r)));
    v[1] = to_f32(__builtin_bit_cast(T, static_cast<uint16_t>(r >> 16)));
  }
}
template <typename T, int VC> __device__ __forceinline__ Word<T, VC> narrow(const float (&v)[VC]) {
  if constexpr (VC == 1) {
    return __builtin_bit_cast(Word<T, VC>, from_f32<T>(v[0]));
  } else if constexpr (std::is_same_v<T, bf16>) {
    return pack_bf16x2(v[0], v[1]);
  } else {
    return static_cast<uint32_t>(__builtin_bit_cast(uint16_t, from_f32<T>(v[0]))) |
           static_cast<uint32_t>(__builtin_bit_cast(uint16_t, from_f32<T>(v[1]))) << 16;
  }
}

// ---- gates -----------------------------------------------------------------------------
// The exponentials are v_exp_f32's: for a gate x it is off by |x| 2^-24 at
// most, and errors of neighbouring steps are independent, so they do not add
// up over the decay's memory; a systematic error would (a = exp(-s) near 1 and
// q are therefore formed from s, whose own error is relative).

__device__ __forceinline__ float gate(float x, float& e) {
  e = fast_exp(-x);
  return fast_rcp(1.0f + e);
}
// 1 - sigmoid from the sigmoid's exponential; an infinite one is cut, so that
// it gives 0 beside a sigmoid of 0 (whose product is wanted) and not NaN.
__device__ __forceinline__ float rest(float e, float sigmoid) { return fminf(e, 3e38f) * sigmoid; }

// q = 1 - exp(-2 s) for s >= 0, given a = exp(-s): below 2 s = 1/2 by a
// polynomial of (1 - exp(-y)) / y (degree 5, fitted to 1.3e-9), above it by
// the difference, which loses little more than a bit.
__device__ __forceinline__ float input_share(float s, float a) {
  const float y = 2.0f * s;
  float q = -0.001124026020988822f;
  q = fmaf(q, y, 0.008190391585230827f);
  q = fmaf(q, y, -0.04163041338324547f);
  q = fmaf(q, y, 0.16666248440742493f);
  q = fmaf(q, y, -0.4999998211860657f);
  q = fmaf(q, y, 1.0f);
  return y < 0.5f ? q * y : fmaf(-a, a, 1.0f);
}

// ---- a workgroup's place ------------------------------------------------------------------

struct Place {
  int lane, w;
  int64_t b, split, d;  // first channel of the lane
  int64_t t0, t1;       // steps of the split
  bool live;
  int64_t dd;           // d, or 0 for lanes beyond the last channel
};
template <int VC> __device__ __forceinline__ Place place(const GatedScanParams& p, int64_t splits) {
  Place q;
  q.lane = threadIdx.x & 63;
  q.w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t tiles = (p.dim + 64 * VC - 1) / (64 * VC);
  const int64_t row = blockIdx.x / tiles;
  q.b = row / splits;
  q.split = row % splits;
  q.d = ((blockIdx.x % tiles) * 64 + q.lane) * VC;
  q.live = q.d < p.dim;
  q.dd = q.live ? q.d : 0;
  q.t0 = q.split * p.split_len;
  q.t1 = q.t0 + p.split_len < p.len ? q.t0 + p.split_len : p.len;
  return q;
}

template <typename T, int VC> struct Column {
  const char* base;
  int64_t step;
  __device__ __forceinline__ Column(const void* ptr, const int64_t (&s)[3], const Place& q)
      : base(static_cast<const char*>(ptr) + (q.b * s[0] + q.dd * s[2]) * static_cast<int64_t>(sizeof(T))),
        step(s[1] * static_cast<int64_t>(sizeof(T))) {}
  __device__ __forceinline__ Word<T, VC> load(int64_t t) const {
    return *reinterpret_cast<const Word<T, VC>*>(base + t * step);
  }
  __device__ __forceinline__ void store(int64_t t, const float (&v)[VC]) const {
    *reinterpret_cast<Word<T, VC>*>(const_cast<char*>(base) + t * step) = narrow<T, VC>(v);
  }
};

// Bit i: step ts + i starts another sequence than the step before it.
__device__ __forceinline__ uint64_t starts(const GatedScanParams& p, const Place& q, int64_t ts) {
  if (p.seq_idx == nullptr) return 0;
  const int64_t t = ts + q.lane;
  const int32_t* ids = p.seq_idx + q.b * p.len;
  bool s = false;
  if (q.lane < TS && t > 0 && t < p.len) s = ids[t] != ids[t - 1];
  return __ballot(s);
}

// ---- forward -----------------------------------------------------------------------------
// SUM: the split's (P, S) only, for the splits that others start from.

template <typename T, int VC, bool SUM>
__global__ __launch_bounds__(64 * W) void gated_fwd_kernel(const GatedScanParams p) {
  const Place q = place<VC>(p, SUM ? p.nsplit - 1 : p.nsplit);
  const Column<T, VC> x(p.x, p.sx, q), ag(p.a_gate, p.sa, q), ig(p.x_gate, p.si, q), y(p.y, p.sy, q);
  const int64_t nseg = (p.len + TS - 1) / TS;
  __shared__ float2 agg[2][W][64 * VC];
  float csp[VC], carry[VC], run[VC];  // run: the product of the decays so far (SUM)
#pragma unroll
  for (int v = 0; v < VC; ++v) {
    csp[v] = p.c * softplus_acc(p.decay[q.dd + v]);
    carry[v] = SUM || p.init == nullptr ? 0.f : p.init[q.b * p.dim + q.dd + v];
    run[v] = 1.f;
  }
  if constexpr (!SUM) {
    for (int64_t sp = 0; sp < q.split; ++sp)
#pragma unroll
      for (int v = 0; v < VC; ++v) {
        const float2 s = p.sums[(q.b * p.nsplit + sp) * p.dim + q.dd + v];
        carry[v] = fmaf(s.x, carry[v], s.y);
      }
  }
  Word<T, VC> rx[TS], ra[TS], ri[TS];
  auto fetch = [&](int64_t ts) {
#pragma unroll
    for (int i = 0; i < TS; ++i) {
      const int64_t t = ts + i < q.t1 ? ts + i : q.t1 - 1;
      ra[i] = ag.load(t);
      ri[i] = ig.load(t);
      rx[i] = x.load(t);
    }
  };
  int buf = 0;
  if (q.t0 < q.t1) fetch(q.t0 + q.w * TS);
  for (int64_t t0 = q.t0; t0 < q.t1; t0 += kGatedChunk, buf ^= 1) {
    const int64_t ts = t0 + q.w * TS;
    const int n = static_cast<int>(q.t1 - ts < 0 ? 0 : q.t1 - ts < TS ? q.t1 - ts : TS);
    const uint64_t cut = starts(p, q, ts);
    float a[TS][VC], u[TS][VC], P[VC], S[VC];
#pragma unroll
    for (int v = 0; v < VC; ++v) {
      P[v] = 1.f;
      S[v] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < TS; ++i) {
      float fx[VC], fa[VC], fi[VC];
      widen<T, VC>(rx[i], fx);
      widen<T, VC>(ra[i], fa);
      widen<T, VC>(ri[i], fi);
#pragma unroll
      for (int v = 0; v < VC; ++v) {
        float e;
        const float s = csp[v] * gate(fa[v], e);
        const float dec = fast_exp(-s);
        const float m = __builtin_amdgcn_sqrtf(input_share(s, dec));
        a[i][v] = i < n ? (((cut >> i) & 1) != 0 ? 0.f : dec) : 1.f;
        u[i][v] = i < n ? m * gate(fi[v], e) * fx[v] : 0.f;
        S[v] = fmaf(a[i][v], S[v], u[i][v]);
        P[v] *= a[i][v];
      }
    }
    if (t0 + kGatedChunk < q.t1) fetch(ts + kGatedChunk);
#pragma unroll
    for (int v = 0; v < VC; ++v) agg[buf][q.w][v * 64 + q.lane] = make_float2(P[v], S[v]);
    __syncthreads();
    float h[VC];
#pragma unroll
    for (int v = 0; v < VC; ++v) h[v] = carry[v];
#pragma unroll
    for (int o = 0; o < W; ++o)
#pragma unroll
      for (int v = 0; v < VC; ++v) {
        if (o == q.w) h[v] = carry[v];
        const float2 s = agg[buf][o][v * 64 + q.lane];
        carry[v] = fmaf(s.x, carry[v], s.y);
        if constexpr (SUM) run[v] *= s.x;
      }
    if constexpr (!SUM) {
      if (q.live && n > 0) {
        if (p.ckpt != nullptr) {
          float* to = p.ckpt + (q.b * nseg + ts / TS) * p.dim + q.d;
#pragma unroll
          for (int v = 0; v < VC; ++v) to[v] = h[v];
        }
#pragma unroll
        for (int i = 0; i < TS; ++i) {
#pragma unroll
          for (int v = 0; v < VC; ++v) h[v] = fmaf(a[i][v], h[v], u[i][v]);
          if (i < n) y.store(ts + i, h);
        }
      }
    }
  }
  if (q.live && q.w == 0) {
#pragma unroll
    for (int v = 0; v < VC; ++v) {
      if constexpr (SUM) p.sums[(q.b * p.nsplit + q.split) * p.dim + q.d + v] = make_float2(run[v], carry[v]);
      else if (p.last != nullptr && q.split == p.nsplit - 1) p.last[q.b * p.dim + q.d + v] = carry[v];
    }
  }
}

// ---- backward ----------------------------------------------------------------------------

// (P, S) of the gradient's step over a split, from its last step to its first,
// for every split but the first. Its S is what leaves the split to the left
// when nothing enters from the right.
template <typename T, int VC>
__global__ __launch_bounds__(64 * W) void gated_bwd_sum_kernel(const GatedScanParams p) {
  Place q = place<VC>(p, p.nsplit - 1);
  q.split += 1;
  q.t0 = q.split * p.split_len;
  q.t1 = q.t0 + p.split_len < p.len ? q.t0 + p.split_len : p.len;
  const Column<T, VC> ag(p.a_gate, p.sa, q), dy(p.dy, p.sdy, q);
  __shared__ float2 agg[2][W][64 * VC];
  float csp[VC], carry[VC], run[VC];
#pragma unroll
  for (int v = 0; v < VC; ++v) {
    csp[v] = p.c * softplus_acc(p.decay[q.dd + v]);
    carry[v] = 0.f;
    run[v] = 1.f;
  }
  int buf = 0;
  const int64_t chunks = (q.t1 - q.t0 + kGatedChunk - 1) / kGatedChunk;
  for (int64_t ch = chunks - 1; ch >= 0; --ch, buf ^= 1) {
    const int64_t ts = q.t0 + ch * kGatedChunk + q.w * TS;
    const int n = static_cast<int>(q.t1 - ts < 0 ? 0 : q.t1 - ts < TS ? q.t1 - ts : TS);
    const uint64_t cut = starts(p, q, ts);
    Word<T, VC> ra[TS], rd[TS];
#pragma unroll
    for (int i = 0; i < TS; ++i) {
      const int64_t t = ts + i < q.t1 ? ts + i : q.t1 - 1;
      ra[i] = ag.load(t);
      rd[i] = dy.load(t);
    }
    float P[VC], S[VC];
#pragma unroll
    for (int v = 0; v < VC; ++v) {
      P[v] = 1.f;
      S[v] = 0.f;
    }
#pragma unroll
    for (int i = TS - 1; i >= 0; --i) {
      float fa[VC], fd[VC];
      widen<T, VC>(ra[i], fa);
      widen<T, VC>(rd[i], fd);
#pragma unroll
      for (int v = 0; v < VC; ++v) {
        float e;
        const float dec = fast_exp(-csp[v] * gate(fa[v], e));
        const float ka = i < n ? (((cut >> i) & 1) != 0 ? 0.f : dec) : 1.f;
        S[v] = ka * (S[v] + (i < n ? fd[v] : 0.f));
        P[v] *= ka;
      }
    }
#pragma unroll
    for (int v = 0; v < VC; ++v) agg[buf][q.w][v * 64 + q.lane] = make_float2(P[v], S[v]);
    __syncthreads();
#pragma unroll
    for (int o = W - 1; o >= 0; --o)
#pragma unroll
      for (int v = 0; v < VC; ++v) {
        const float2 s = agg[buf][o][v * 64 + q.lane];
        carry[v] = fmaf(s.x, carry[v], s.y);
        run[v] *= s.x;
      }
  }
  if (q.live && q.w == 0)
#pragma unroll
    for (int v = 0; v < VC; ++v)
      p.sums[(q.b * p.nsplit + q.split) * p.dim + q.d + v] = make_float2(run[v], carry[v]);
}

template <typename T, int VC>
__global__ __launch_bounds__(64 * W) void gated_bwd_kernel(const GatedScanParams p) {
  // 1 - rho and 1 - iota to their own ulp are kept for float32 gradients; a
  // 16-bit one does not show the difference to 1 minus the sigmoid.
  constexpr bool EXACT = sizeof(T) == 4;
  const Place q = place<VC>(p, p.nsplit);
  const Column<T, VC> x(p.x, p.sx, q), ag(p.a_gate, p.sa, q), ig(p.x_gate, p.si, q), dy(p.dy, p.sdy, q);
  const Column<T, VC> dx(p.dx, p.sdx, q), da(p.da_gate, p.sda, q), di(p.dx_gate, p.sdi, q);
  const int64_t nseg = (p.len + TS - 1) / TS;
  __shared__ float2 agg[2][W][64 * VC];
  float csp[VC], carry[VC], acc[VC];  // acc: this lane's sum of e rho
#pragma unroll
  for (int v = 0; v < VC; ++v) {
    csp[v] = p.c * softplus_acc(p.decay[q.dd + v]);
    carry[v] = p.dlast == nullptr ? 0.f : p.dlast[q.b * p.dim + q.dd + v];
    acc[v] = 0.f;
  }
  for (int64_t sp = p.nsplit - 1; sp > q.split; --sp)
#pragma unroll
    for (int v = 0; v < VC; ++v) {
      const float2 s = p.sums[(q.b * p.nsplit + sp) * p.dim + q.dd + v];
      carry[v] = fmaf(s.x, carry[v], s.y);
    }
  int buf = 0;
  const int64_t chunks = q.t1 > q.t0 ? (q.t1 - q.t0 + kGatedChunk - 1) / kGatedChunk : 0;
  for (int64_t ch = chunks - 1; ch >= 0; --ch, buf ^= 1) {
    const int64_t ts = q.t0 + ch * kGatedChunk + q.w * TS;
    const int n = static_cast<int>(q.t1 - ts < 0 ? 0 : q.t1 - ts < TS ? q.t1 - ts : TS);
    const uint64_t cut = starts(p, q, ts);
    Word<T, VC> rx[TS], ra[TS], ri[TS], rd[TS];
    float h[VC];
#pragma unroll
    for (int i = 0; i < TS; ++i) {
      const int64_t t = ts + i < q.t1 ? ts + i : q.t1 - 1;
      ra[i] = ag.load(t);
      ri[i] = ig.load(t);
      rx[i] = x.load(t);
      rd[i] = dy.load(t);
    }
#pragma unroll
    for (int v = 0; v < VC; ++v) h[v] = n > 0 ? p.ckpt[(q.b * nseg + ts / TS) * p.dim + q.dd + v] : 0.f;
    float rho[TS][VC], iota[TS][VC], share[TS][VC], ka[TS][VC], kah[TS][VC];
    float nrho[EXACT ? TS : 1][VC], niota[EXACT ? TS : 1][VC];
    float P[VC], S[VC];
#pragma unroll
    for (int v = 0; v < VC; ++v) {
      P[v] = 1.f;
      S[v] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < TS; ++i) {
      float fx[VC], fa[VC], fi[VC];
      widen<T, VC>(rx[i], fx);
      widen<T, VC>(ra[i], fa);
      widen<T, VC>(ri[i], fi);
#pragma unroll
      for (int v = 0; v < VC; ++v) {
        float ea, ei;
        rho[i][v] = gate(fa[v], ea);
        iota[i][v] = gate(fi[v], ei);
        if constexpr (EXACT) {
          nrho[i][v] = rest(ea, rho[i][v]);
          niota[i][v] = rest(ei, iota[i][v]);
        }
        const float s = csp[v] * rho[i][v];
        const float dec = fast_exp(-s);
        share[i][v] = input_share(s, dec);
        ka[i][v] = i < n ? (((cut >> i) & 1) != 0 ? 0.f : dec) : 1.f;
        kah[i][v] = ka[i][v] * h[v];
        h[v] = fmaf(__builtin_amdgcn_sqrtf(share[i][v]) * iota[i][v], fx[v], kah[i][v]);
        P[v] *= ka[i][v];
      }
    }
#pragma unroll
    for (int i = TS - 1; i >= 0; --i) {
      float fd[VC];
      widen<T, VC>(rd[i], fd);
#pragma unroll
      for (int v = 0; v < VC; ++v) S[v] = ka[i][v] * (S[v] + (i < n ? fd[v] : 0.f));
    }
#pragma unroll
    for (int v = 0; v < VC; ++v) agg[buf][q.w][v * 64 + q.lane] = make_float2(P[v], S[v]);
    __syncthreads();
    float G[VC];
#pragma unroll
    for (int v = 0; v < VC; ++v) G[v] = carry[v];
#pragma unroll
    for (int o = W - 1; o >= 0; --o)
#pragma unroll
      for (int v = 0; v < VC; ++v) {
        if (o == q.w) G[v] = carry[v];
        const float2 s = agg[buf][o][v * 64 + q.lane];
        carry[v] = fmaf(s.x, carry[v], s.y);
      }
#pragma unroll
    for (int i = TS - 1; i >= 0; --i) {
      if (i >= n) continue;
      float fx[VC], fd[VC], ox[VC], oa[VC], oi[VC];
      widen<T, VC>(rx[i], fx);
      widen<T, VC>(rd[i], fd);
#pragma unroll
      for (int v = 0; v < VC; ++v) {
        const float g = fd[v] + G[v];
        // 1 / m, cut above what the smallest normal q gives: a closed gate
        // (q = 0) has m = 0, and a^2 s / m = 0, which is its limit.
        const float inv = fminf(__builtin_amdgcn_rsqf(share[i][v]), 1e19f);
        const float gi = g * iota[i][v];
        ox[v] = gi * (share[i][v] * inv);
        oi[v] = ox[v] * fx[v] * (EXACT ? niota[EXACT ? i : 0][v] : 1.0f - iota[i][v]);
        const float e = fmaf(gi * fx[v], (1.0f - share[i][v]) * inv, -g * kah[i][v]);
        oa[v] = e * (csp[v] * rho[i][v]) * (EXACT ? nrho[EXACT ? i : 0][v] : 1.0f - rho[i][v]);
        acc[v] = fmaf(e, rho[i][v], acc[v]);
        G[v] = ka[i][v] * g;
      }
      if (q.live) {
        dx.store(ts + i, ox);
        di.store(ts + i, oi);
        da.store(ts + i, oa);
      }
    }
  }
  if (q.live && q.w == 0 && q.split == 0 && p.dinit != nullptr)
#pragma unroll
    for (int v = 0; v < VC; ++v) p.dinit[q.b * p.dim + q.d + v] = carry[v];
  __syncthreads();
#pragma unroll
  for (int v = 0; v < VC; ++v) agg[0][q.w][v * 64 + q.lane].x = acc[v];
  __syncthreads();
  if (q.w == 0 && q.live)
#pragma unroll
    for (int v = 0; v < VC; ++v) {
      float sum = 0.f, e;
      for (int o = 0; o < W; ++o) sum += agg[0][o][v * 64 + q.lane].x;
      p.ddecay_part[(q.b * p.nsplit + q.split) * p.dim + q.d + v] = sum * p.c * gate(p.decay[q.d + v], e);
    }
}

// ddecay: the partial sums of the batch rows and splits, added in order.
__global__ __launch_bounds__(64) void gated_ddecay_kernel(const GatedScanParams p) {
  const int64_t d = blockIdx.x * 64ll + threadIdx.x;
  if (d >= p.dim) return;
  float sum = 0.f;
#pragma unroll 8
  for (int64_t k = 0; k < p.batch * p.nsplit; ++k) sum += p.ddecay_part[k * p.dim + d];
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
  float e;
  const float s = p.c * softplus_acc(p.decay[d]) * gate(ld<T>(p.a_gate, b * p.sa[0] + d * p.sa[1]), e);
  const float a = fast_exp(-s);
  const float in = __builtin_amdgcn_sqrtf(input_share(s, a)) * gate(ld<T>(p.x_gate, b * p.si[0] + d * p.si[1]), e);
  float* h = p.state + row * p.sst[0] + d * p.sst[1];
  const float v = fmaf(a, *h, in * ld<T>(p.x, b * p.sx[0] + d * p.sx[1]));
  *h = v;
  *y = from_f32<T>(v);
}

template <typename F> void by_dtype(int dtype, F&& f) {
  if (dtype == MCPU_F32) f(float{});
  else if (dtype == MCPU_BF16) f(bf16{});
  else f(f16{});
}

template <typename T, int VC> void launch_fwd(const GatedScanParams& p, hipStream_t st) {
  const int64_t tiles = (p.dim + 64 * VC - 1) / (64 * VC);
  if (p.nsplit > 1)
    hipLaunchKernelGGL((gated_fwd_kernel<T, VC, true>), dim3(static_cast<unsigned>(tiles * p.batch * (p.nsplit - 1))),
                       dim3(64 * W), 0, st, p);
  hipLaunchKernelGGL((gated_fwd_kernel<T, VC, false>), dim3(static_cast<unsigned>(tiles * p.batch * p.nsplit)),
                     dim3(64 * W), 0, st, p);
}

template <typename T, int VC> void launch_bwd(const GatedScanParams& p, hipStream_t st) {
  const int64_t tiles = (p.dim + 64 * VC - 1) / (64 * VC);
  if (p.nsplit > 1)
    hipLaunchKernelGGL((gated_bwd_sum_kernel<T, VC>), dim3(static_cast<unsigned>(tiles * p.batch * (p.nsplit - 1))),
                       dim3(64 * W), 0, st, p);
  hipLaunchKernelGGL((gated_bwd_kernel<T, VC>), dim3(static_cast<unsigned>(tiles * p.batch * p.nsplit)), dim3(64 * W),
                     0, st, p);
}

}  // namespace

void gated_scan_plan(GatedScanParams& p, int vec) {
  p.vec = vec;
  const int64_t wgs = (p.dim + 64 * vec - 1) / (64 * vec) * p.batch;
  const int64_t chunks = (p.len + kGatedChunk - 1) / kGatedChunk;
  int64_t n = wgs >= 400 || wgs < 1 ? 1 : (1024 + wgs - 1) / wgs;
  if (n > chunks) n = chunks;
  if (n < 1) n = 1;
  const int64_t per = (chunks + n - 1) / n;  // chunks per split
  p.split_len = (per < 1 ? 1 : per) * kGatedChunk;
  p.nsplit = chunks < 1 ? 1 : (chunks + per - 1) / per;
}

hipError_t gated_scan_fwd_launch(const GatedScanParams& p, int dtype, hipStream_t st) {
  by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    if constexpr (sizeof(T) == 2) {
      if (p.vec == 2) return launch_fwd<T, 2>(p, st);
    }
    launch_fwd<T, 1>(p, st);
  });
  return hipGetLastError();
}

hipError_t gated_scan_bwd_launch(const GatedScanParams& p, int dtype, hipStream_t st) {
  by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    if constexpr (sizeof(T) == 2) {
      if (p.vec == 2) return launch_bwd<T, 2>(p, st);
    }
    launch_bwd<T, 1>(p, st);
  });
  hipLaunchKernelGGL(gated_ddecay_kernel, dim3(static_cast<unsigned>((p.dim + 63) / 64)), dim3(64), 0, st, p);
  return hipGetLastError();
}

hipError_t gated_step_launch(const GatedStepParams& p, int dtype, hipStream_t st) {
  const unsigned grid = static_cast<unsigned>((p.batch * p.dim + 255) / 256);
  by_dtype(dtype, [&](auto t) {
    hipLaunchKernelGGL(gated_step_kernel<decltype(t)>, dim3(grid), dim3(256), 0, st, p);
  });
  return hipGetLastError();
}

}  // namespace mcpu
