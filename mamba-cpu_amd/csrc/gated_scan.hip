// Gated linear recurrence on gfx950: forward, backward and the single-token
// step. Per batch row, step t and channel d, all in float32:
//
//   rho = sigmoid(a_gate)   iota = sigmoid(x_gate)   s = c softplus(decay_d) rho
//   a = exp(-s)             m = sqrt(q), q = 1 - exp(-2 s)
//   h_t = k_t a h_{t-1} + m iota x_t,   y_t = h_t
//
// with k_t = 0 at the first step of another sequence of a packed row, else 1.
// The step h -> a h + b composes as (P, S): h -> P h + S, so time is split: a
// wave takes kGatedT = 16 consecutive steps of 64 channels in registers and forms
// their (P, S), the workgroup's waves exchange theirs through LDS, and each
// wave then knows the state in front of its segment, given the one in front of
// the workgroup's chunk.
//
// A workgroup takes one chunk (128 steps forward, 64 backward) of 64 channels, so
// that every length fills the chip and every input is read once. The state in
// front of a chunk comes from the chunks before it: a workgroup publishes its
// (P, S) as soon as it has them (its inputs stay in registers), then looks back,
// a predecessor per wave, until nothing older matters: a predecessor that knows
// the state behind its chunk has published that, as (0, h), in the place of its
// (P, S). Its own (0, h) is published before its outputs are written.
// Every wait ends: the chunks of a row's tile are taken by ticket, in the order
// of time, so the chunks a workgroup waits for have been taken by workgroups
// that run or have ended, and a workgroup publishes its (P, S) before it waits.
// Records pass between workgroups as single 64-bit words, written by agent-scope
// atomic stores and polled by agent-scope atomic loads; a word carries all that
// is read, and either of a chunk's two is right, so no fence is needed.
//
// Bound: the inputs and outputs once, for 8 x 2048 x 1536 bf16 201 MB forward
// and 352 MB backward, and vector issue: 43 and 65 instructions a step and
// channel. Measured there: forward 57 us (3.5 TB/s), backward 87 us (4.0 TB/s), a
// training step with its clears and the decay's sum 148 us. Other splits, for the
// same step:
//   two launches a direction, the first for every split's (P, S)   221 us
//   8 steps a wave: twice the segments, each with its exchange and
//   look back, which are 20 instructions a step then               166 us
//   workgroups that stay and take chunk after chunk, the next one's
//   inputs requested ahead: the chain of a tile gets longer        276 us
// What is left is that chain, the time from a chunk's inputs to its (0, h), and
// that loads, arithmetic and the wait of one workgroup overlap with only three
// others' on a CU.
//
// Backward, with g_t = dL/dh_t:  g_t = dy_t + k_{t+1} a_{t+1} g_{t+1},
//   dx = g m iota          dx_gate = dx x (1 - iota)
//   e  = g (iota x a^2 / m - k a h_{t-1})
//   da_gate = e s (1 - rho)       ddecay = sum e c rho sigmoid(decay)
// is the same scan from the other end; the states it needs are recomputed
// from the one the forward kept in front of every segment, in float32 (the
// stored y may be 16 bits wide).
#include "gated_scan.h"
#include "launch.h"
#include "lm_math.h"

namespace mcpu {
namespace {

constexpr int TS = kGatedT;

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
// polynomial of (1 - exp(-y)) / y, y = 2 s (degree 5, within 4.2e-9; here in
// powers of s), above it by the difference, which loses little more than a bit.
__device__ __forceinline__ float input_share(float s, float a) {
  float q = -64 * 0.001124026020988822f;
  q = fmaf(q, s, 32 * 0.008190391585230827f);
  q = fmaf(q, s, -16 * 0.04163041338324547f);
  q = fmaf(q, s, 8 * 0.16666248440742493f);
  q = fmaf(q, s, -4 * 0.4999998211860657f);
  q = fmaf(q, s, 2.0f);
  return s < 0.25f ? q * s : fmaf(-a, a, 1.0f);
}

// ---- a workgroup's place ------------------------------------------------------------------

struct Place {
  int lane, w;
  int64_t b, chunk, d;  // d: the lane's channel
  int64_t ts;           // first step of the wave's segment
  int n;                // steps of the segment
  bool live;
  int64_t dd;           // d, or the tile's first channel for lanes beyond the last
};
// Which chunk of its row's tile the workgroup takes: the next one in the order of
// time, from the last on with LAST_FIRST. A counter for each tile: when thousands
// of workgroups share one, each waits 1.4 us for it, 5 us at the start.
template <int W, bool LAST_FIRST> __device__ __forceinline__ Place place(const GatedScanParams& p) {
  __shared__ uint32_t ticket;
  Place q;
  q.lane = threadIdx.x & 63;
  q.w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t tiles = static_cast<uint32_t>((p.dim + 63) / 64);
  const uint32_t rows = tiles * static_cast<uint32_t>(p.batch), row = (static_cast<uint32_t>(p.first) + blockIdx.x) % rows;
  uint32_t t = 0;
  if (p.chunks > 1) {
    if (threadIdx.x == 0) ticket = atomicAdd(p.tickets + row, 1u);
    __syncthreads();
    t = __builtin_amdgcn_readfirstlane(ticket);
  }
  q.chunk = LAST_FIRST ? p.chunks - 1 - t : t;
  q.b = row / tiles;
  const int64_t first = row % tiles * 64ll;
  q.d = first + q.lane;
  q.live = q.d < p.dim;
  q.dd = q.live ? q.d : first;
  q.ts = (q.chunk * W + q.w) * TS;
  const int64_t left = p.len - q.ts;
  q.n = left < 0 ? 0 : left < TS ? static_cast<int>(left) : TS;
  return q;
}

// The wave's segment of an operand: a scalar base, the lane's byte offset, and
// a scalar offset per step. Steps behind the row's end read its last one.
template <typename T> struct Column {
  __amdgpu_buffer_rsrc_t rsrc;
  uint32_t lane, step;
  __device__ __forceinline__ Column(const void* ptr, const int64_t (&s)[3], const GatedScanParams& p, const Place& q)
      : rsrc(wave_rsrc(static_cast<const char*>(ptr) +
                       (q.b * s[0] + (q.n > 0 ? q.ts : p.len - 1) * s[1]) * static_cast<int64_t>(sizeof(T)))),
        lane(static_cast<uint32_t>(q.dd * s[2] * static_cast<int64_t>(sizeof(T)))),
        step(static_cast<uint32_t>(s[1] * static_cast<int64_t>(sizeof(T)))) {}
  // The bits, to be widened where they are used: that is where the wave waits.
  __device__ __forceinline__ uint32_t load(const Place& q, int i) const {
    const int at = i < q.n ? i : q.n > 0 ? q.n - 1 : 0;
    if constexpr (sizeof(T) == 4) return __builtin_amdgcn_raw_buffer_load_b32(rsrc, lane, at * step, 0);
    else return __builtin_amdgcn_raw_buffer_load_b16(rsrc, lane, at * step, 0);
  }
  __device__ __forceinline__ void store(int i, float v) const {
    if constexpr (sizeof(T) == 4)
      __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, v), rsrc, lane, i * step, 0);
    else
      __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, from_f32<T>(v)), rsrc, lane, i * step, 0);
  }
};
template <typename T> __device__ __forceinline__ float widen(uint32_t bits) {
  if constexpr (sizeof(T) == 4) return __builtin_bit_cast(float, bits);
  else return to_f32(__builtin_bit_cast(T, static_cast<uint16_t>(bits)));
}

// Bit i: step ts + i starts another sequence than the step before it.
__device__ __forceinline__ uint32_t starts(const GatedScanParams& p, const Place& q) {
  const int64_t t = q.ts + q.lane;
  const int32_t* ids = p.seq_idx + q.b * p.len;
  bool s = false;
  if (q.lane < TS && t > 0 && t < p.len) s = ids[t] != ids[t - 1];
  return static_cast<uint32_t>(__ballot(s));
}

// ---- steps and what is published of them --------------------------------------------------

// P is 0 where a sequence starts among the steps, and only there: products of
// decays are held above 0, so that a NaN or an infinity stays in the state of
// its sequence however much decays, and never enters the next one's. The smallest
// they take is the smallest float32 number (a denormal; the kernels are built with
// them), so that a state leaves a segment or chunk at most 2^-149 of itself too large.
constexpr float kFaint = 0x1p-149f;
__device__ __forceinline__ float after(float2 s, float h) { return s.x == 0.f ? s.y : fmaf(s.x, h, s.y); }
__device__ __forceinline__ float join(float P, float Q) { return fmaxf(P * Q, fminf(fminf(P, Q), kFaint)); }

// A record is (P, S) with every bit flipped, so that zeroed memory, the flipped
// all-ones NaN pair, means none yet; a NaN is published as another one.
__device__ __forceinline__ uint32_t plain(float x) { return x == x ? __builtin_bit_cast(uint32_t, x) : 0x7fc00000u; }
__device__ __forceinline__ void publish(uint64_t* at, float P, float S) {
  const uint64_t v = ~(static_cast<uint64_t>(plain(P)) << 32 | plain(S));
  __hip_atomic_store(at, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ uint64_t peek(const uint64_t* at) {
  return __hip_atomic_load(at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

constexpr int kWindows = 4;  // windows of W chunks that are kept
template <int W> struct Exchange {
  float2 agg[W][64];                // the segments' (P, S)
  float2 win[kWindows + 2][W][64];  // what the waves found of W neighbouring chunks; two for those further back
};

// The state that enters the wave's segment, from the segments' (P, S) and
// `edge`, the state that enters the row's first chunk (in the direction of the
// scan: DIR 1 forward, -1 backward). `out` is the state behind the chunk.
template <int W, int DIR>
__device__ __forceinline__ void scan_chunks(const GatedScanParams& p, const Place& q, Exchange<W>& x, float P, float S,
                                            float edge, float& in, float& out) {
  x.agg[q.w][q.lane] = make_float2(P, S);
  __syncthreads();
  // The segments before this one, and the whole chunk.
  float2 mine, all = make_float2(1.f, 0.f);
#pragma unroll
  for (int o = 0; o < W; ++o) {
    const int seg = DIR > 0 ? o : W - 1 - o;
    if (seg == q.w) mine = all;
    const float2 s = x.agg[seg][q.lane];
    all = make_float2(join(all.x, s.x), after(s, all.y));
  }
  const int64_t first = DIR > 0 ? 0 : p.chunks - 1;
  const int64_t back = DIR * (q.chunk - first);  // chunks before this one
  uint64_t* const rec = p.records + q.b * p.chunks * p.dim + q.dd;
  float state = edge;
  if (back > 0) {
    if (q.w == 0 && q.live) publish(rec + q.chunk * p.dim, all.x, all.y);
    auto slot = [](int64_t win) {
      return win < kWindows ? static_cast<int>(win) : kWindows + static_cast<int>(win & 1);
    };
    // This wave's chunk of a window, as published.
    auto fetch = [&](int64_t win) {
      const int64_t away = win * W + q.w + 1;  // how far back the chunk is
      // In front of the row's first chunk: the edge, then nothing.
      float2 s = away == back + 1 ? make_float2(0.f, edge) : make_float2(1.f, 0.f);
      if (away <= back) {
        const uint64_t* at = rec + (q.chunk - DIR * away) * p.dim;
        uint64_t word = peek(at);
        while (__ballot(word == 0) != 0) {
          __builtin_amdgcn_s_sleep(1);
          word = peek(at);
        }
        s.x = __builtin_bit_cast(float, ~static_cast<uint32_t>(word >> 32));
        s.y = __builtin_bit_cast(float, ~static_cast<uint32_t>(word));
      }
      x.win[slot(win)][q.w][q.lane] = s;
      __syncthreads();
    };
    // Back until every channel has met a chunk that does not depend on older ones.
    bool known = false;
    int64_t win = 0;
    for (;; ++win) {
      fetch(win);
#pragma unroll
      for (int o = 0; o < W; ++o) known |= x.win[slot(win)][o][q.lane].x == 0.f;
      // All waves read the same values, so all leave together.
      if (__ballot(!known) == 0 || (win + 1) * W > back) break;
    }
    // Then forward again, one chunk after the other: the state behind chunk j is
    // always after((P, S)_j, the state in front of it), whether another
    // workgroup formed it or this one, so that the result does not depend on
    // what had been published when. Windows further back than those kept are
    // read again, except the last.
    state = 0.f;
    for (int64_t w = win; w >= 0; --w) {
      if (w >= kWindows && w < win) fetch(w);
#pragma unroll
      for (int o = W - 1; o >= 0; --o) state = after(x.win[slot(w)][o][q.lane], state);
    }
  }
  in = after(mine, state);
  out = after(all, state);
  if (back < p.chunks - 1 && q.w == 0 && q.live) publish(rec + q.chunk * p.dim, 0.f, out);
}

// ---- forward -----------------------------------------------------------------------------
// SEQ: packed sequences.

template <typename T, bool SEQ>
__global__ __launch_bounds__(64 * kGatedFwdWaves) void gated_fwd_kernel(const GatedScanParams p) {
  constexpr int W = kGatedFwdWaves;
  __shared__ Exchange<W> exchange;
  const Place q = place<W, false>(p);
  const Column<T> x(p.x, p.sx, p, q), ag(p.a_gate, p.sa, p, q), ig(p.x_gate, p.si, p, q), y(p.y, p.sy, p, q);
  uint32_t rx[TS], ra[TS], ri[TS];
#pragma unroll
  for (int i = 0; i < TS; ++i) {
    ra[i] = ag.load(q, i);
    ri[i] = ig.load(q, i);
    rx[i] = x.load(q, i);
  }
  const uint32_t cut = SEQ ? starts(p, q) : 0;
  const float csp = p.c * softplus_acc(p.decay[q.dd]);
  const float edge = p.init == nullptr ? 0.f : p.init[q.b * p.dim + q.dd];
  float a[TS], u[TS], P = 1.f, S = 0.f;
#pragma unroll
  for (int i = 0; i < TS; ++i) {
    float e;
    const float s = csp * gate(widen<T>(ra[i]), e);
    a[i] = fast_exp(-s);
    u[i] = __builtin_amdgcn_sqrtf(input_share(s, a[i])) * gate(widen<T>(ri[i]), e) * widen<T>(rx[i]);
  }
  // What few segments need is done behind branches that a wave takes as one.
  if (q.n < TS) {
#pragma unroll
    for (int i = 0; i < TS; ++i) {
      a[i] = i < q.n ? a[i] : 1.f;
      u[i] = i < q.n ? u[i] : 0.f;
    }
  }
  // h through the segment, with each(i) behind step i.
  auto walk = [&](float& h, auto&& each) {
    auto steps = [&](auto packed) {
#pragma unroll
      for (int i = 0; i < TS; ++i) {
        h = packed.value && ((cut >> i) & 1) != 0 ? u[i] : fmaf(a[i], h, u[i]);
        each(i);
      }
    };
    if (SEQ && cut != 0) steps(std::true_type{});
    else steps(std::false_type{});
  };
  walk(S, [&](int i) { P *= a[i]; });
  P = cut != 0 ? 0.f : fmaxf(P, kFaint);  // a NaN in P is one in S, too
  float h, out;
  scan_chunks<W, 1>(p, q, exchange, P, S, edge, h, out);
  if (!q.live) return;
  if (q.w == 0 && q.chunk == p.chunks - 1 && p.last != nullptr) p.last[q.b * p.dim + q.d] = out;
  if (q.n <= 0) return;
  if (p.ckpt != nullptr) p.ckpt[(q.b * ((p.len + TS - 1) / TS) + q.ts / TS) * p.dim + q.d] = h;
  walk(h, [&](int i) {
    if (i < q.n) y.store(i, h);
  });
}

// ---- backward ----------------------------------------------------------------------------

template <typename T, bool SEQ>
__global__ __launch_bounds__(64 * kGatedBwdWaves, 4) void gated_bwd_kernel(const GatedScanParams p) {
  constexpr int W = kGatedBwdWaves;
  constexpr bool EXACT = sizeof(T) == 4;
  __shared__ Exchange<W> exchange;
  const Place q = place<W, true>(p);
  const Column<T> x(p.x, p.sx, p, q), ag(p.a_gate, p.sa, p, q), ig(p.x_gate, p.si, p, q), dy(p.dy, p.sdy, p, q);
  uint32_t rx[TS], ra[TS], ri[TS], rd[TS];
#pragma unroll
  for (int i = 0; i < TS; ++i) {
    ra[i] = ag.load(q, i);
    rd[i] = dy.load(q, i);
    ri[i] = ig.load(q, i);
    rx[i] = x.load(q, i);
  }
  const uint32_t cut = SEQ ? starts(p, q) : 0;
  float h = q.n > 0 ? p.ckpt[(q.b * ((p.len + TS - 1) / TS) + q.ts / TS) * p.dim + q.dd] : 0.f;
  const float csp = p.c * softplus_acc(p.decay[q.dd]);
  const float edge = p.dlast == nullptr ? 0.f : p.dlast[q.b * p.dim + q.dd];
  // What a step's gradients are per unit of g: dx, dx_gate, da_gate, e rho; and k a.
  float gx[TS], gi[TS], ga[TS], gd[TS], ka[TS];
#pragma unroll
  for (int i = 0; i < TS; ++i) {
    const bool restart = SEQ && ((cut >> i) & 1) != 0;
    const float fx = widen<T>(rx[i]);
    float ea, ei;
    const float rho = gate(widen<T>(ra[i]), ea), iota = gate(widen<T>(ri[i]), ei);
    const float s = csp * rho;
    const float dec = fast_exp(-s);
    const float share = input_share(s, dec);
    // 1 / m, cut above what the smallest normal share gives: a closed gate
    // (share = 0) has m = 0, and a^2 s / m = 0, which is its limit.
    const float inv = fminf(__builtin_amdgcn_rsqf(share), 1e19f);
    ka[i] = restart ? 0.f : dec;
    const float kah = restart ? 0.f : dec * h;
    gx[i] = iota * (share * inv);
    const float u = gx[i] * fx;
    const float e = fmaf(iota * fx, (1.0f - share) * inv, -kah);
    gd[i] = e * rho;
    // 1 minus a sigmoid to its own ulp for float32 gradients; a 16-bit one
    // does not show the difference.
    gi[i] = EXACT ? u * rest(ei, iota) : fmaf(-u, iota, u);
    ga[i] = EXACT ? e * s * rest(ea, rho) : gd[i] * (csp - s);
    h = kah + u;
    // These five are to be formed here: moved down to their use, their
    // operands would be kept instead, in twice the registers. 128 (the launch
    // bound) leave room for four workgroups a CU.
    asm volatile("" : "+v"(gx[i]), "+v"(gi[i]), "+v"(ga[i]), "+v"(gd[i]), "+v"(ka[i]));
  }
  // 16-bit dy waits two to a register.
  constexpr int PACK = sizeof(T) == 2 ? 2 : 1;
  uint32_t kept[TS / PACK];
#pragma unroll
  for (int i = 0; i < TS; i += PACK) {
    if constexpr (PACK == 2) kept[i / 2] = rd[i] | rd[i + 1] << 16;
    else kept[i] = rd[i];
  }
  auto dy_at = [&](int i) { return widen<T>(kept[i / PACK] >> (PACK == 2 && i % 2 == 1 ? 16 : 0)); };
  float P = 1.f, S = 0.f;
  auto bridge = [&](auto full) {
#pragma unroll
    for (int i = TS - 1; i >= 0; --i) {
      const bool restart = SEQ && ((cut >> i) & 1) != 0, in = full.value || i < q.n;
      ka[i] = in ? ka[i] : 1.f;
      S = restart ? 0.f : ka[i] * (S + (in ? dy_at(i) : 0.f));
      P *= ka[i];
    }
  };
  if (q.n < TS) bridge(std::false_type{});
  else bridge(std::true_type{});
  P = cut != 0 ? 0.f : fmaxf(P, kFaint);
#pragma unroll
  for (int i = 0; i < TS / PACK; ++i) asm volatile("" : "+v"(kept[i]));  // and is not kept widened
  float G, out, acc = 0.f;  // acc: this lane's sum of e rho
  scan_chunks<W, -1>(p, q, exchange, P, S, edge, G, out);
  if (q.live && q.w == 0 && q.chunk == 0 && p.dinit != nullptr) p.dinit[q.b * p.dim + q.d] = out;
  const Column<T> dx(p.dx, p.sdx, p, q), da(p.da_gate, p.sda, p, q), di(p.dx_gate, p.sdi, p, q);
#pragma unroll
  for (int i = TS - 1; i >= 0; --i) {
    if (i >= q.n) continue;
    const float g = dy_at(i) + G;
    acc = fmaf(g, gd[i], acc);
    G = SEQ && ((cut >> i) & 1) != 0 ? 0.f : ka[i] * g;
    if (q.live) {
      dx.store(i, g * gx[i]);
      di.store(i, g * gi[i]);
      da.store(i, g * ga[i]);
    }
  }
  __syncthreads();
  exchange.agg[q.w][q.lane].x = acc;
  __syncthreads();
  if (q.w == 0 && q.live) {
    float sum = 0.f, e;
#pragma unroll
    for (int o = 0; o < W; ++o) sum += exchange.agg[o][q.lane].x;
    p.ddecay_part[(q.b * p.chunks + q.chunk) * p.dim + q.d] = sum * p.c * gate(p.decay[q.d], e);
  }
}

constexpr int kReduceWaves = 16;

// No steps: the state that enters leaves.
__global__ __launch_bounds__(256) void gated_edge_kernel(const float* from, float* to, int64_t n, int64_t first) {
  const int64_t i = (first + blockIdx.x) * 256 + threadIdx.x;
  if (i < n) to[i] = from == nullptr ? 0.f : from[i];
}

// ddecay: every kReduceWaves-th partial sum by one wave, then the waves' in order.
__global__ __launch_bounds__(64 * kReduceWaves) void gated_ddecay_kernel(const GatedScanParams p) {
  __shared__ float sums[kReduceWaves][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t d = (p.first + blockIdx.x) * 64 + lane;
  float sum = 0.f;
  if (d < p.dim) {
#pragma unroll 8
    for (int64_t k = wave; k < p.batch * p.chunks; k += kReduceWaves) sum += p.ddecay_part[k * p.dim + d];
  }
  sums[wave][lane] = sum;
  __syncthreads();
  if (wave > 0 || d >= p.dim) return;
  for (int v = 1; v < kReduceWaves; ++v) sum += sums[v][lane];
  p.ddecay[d] = sum;
}

// One token: state (rows, dim) float32 in place.
template <typename T>
__global__ __launch_bounds__(256) void gated_step_kernel(const GatedStepParams p) {
  const int64_t n = (p.first + blockIdx.x) * 256 + threadIdx.x;
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

}  // namespace

hipError_t gated_edge_launch(const float* from, float* to, int64_t n, hipStream_t st) {
  launch_all((n + 255) / 256, 256, [&](int64_t first, unsigned groups) {
    hipLaunchKernelGGL(gated_edge_kernel, dim3(groups), dim3(256), 0, st, from, to, n, first);
  });
  return hipGetLastError();
}

// A workgroup for each chunk of 64 channels.
static int64_t gated_groups(const GatedScanParams& p) { return (p.dim + 63) / 64 * p.batch * p.chunks; }

hipError_t gated_scan_fwd_launch(GatedScanParams p, int dtype, hipStream_t st) {
  by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    const dim3 block(64 * kGatedFwdWaves);
    launch_all(gated_groups(p), block.x, [&](int64_t first, unsigned groups) {
      p.first = first;
      if (p.seq_idx != nullptr) hipLaunchKernelGGL((gated_fwd_kernel<T, true>), dim3(groups), block, 0, st, p);
      else hipLaunchKernelGGL((gated_fwd_kernel<T, false>), dim3(groups), block, 0, st, p);
    });
  });
  return hipGetLastError();
}

hipError_t gated_scan_bwd_launch(GatedScanParams p, int dtype, hipStream_t st) {
  by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    const dim3 block(64 * kGatedBwdWaves);
    launch_all(gated_groups(p), block.x, [&](int64_t first, unsigned groups) {
      p.first = first;
      if (p.seq_idx != nullptr) hipLaunchKernelGGL((gated_bwd_kernel<T, true>), dim3(groups), block, 0, st, p);
      else hipLaunchKernelGGL((gated_bwd_kernel<T, false>), dim3(groups), block, 0, st, p);
    });
  });
  launch_all((p.dim + 63) / 64, 64 * kReduceWaves, [&](int64_t first, unsigned groups) {
    p.first = first;
    hipLaunchKernelGGL(gated_ddecay_kernel, dim3(groups), dim3(64 * kReduceWaves), 0, st, p);
  });
  return hipGetLastError();
}

hipError_t gated_step_launch(GatedStepParams p, int dtype, hipStream_t st) {
  by_dtype(dtype, [&](auto t) {
    launch_all((p.batch * p.dim + 255) / 256, 256, [&](int64_t first, unsigned groups) {
      p.first = first;
      hipLaunchKernelGGL(gated_step_kernel<decltype(t)>, dim3(groups), dim3(256), 0, st, p);
    });
  });
  return hipGetLastError();
}

}  // namespace mcpu
