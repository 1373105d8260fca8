// The matrix product under the head's losses on gfx950:
//   D(m, n) = sum_k A(m, k) B(n, k)
// for 16-bit operands, accumulated in float32 by v_mfma_f32_32x32x16, a tile of
// 256 x 256 per workgroup of eight waves, 128 x 64 each. An epilogue takes the
// accumulators.
//
// An operand lies either with its terms k side by side ("by row") or with its
// rows m (n) side by side, one term after the other ("by term"); the latter is
// turned on its way out of LDS by ds_read_b64_tr_b16, so that no operand is
// written out transposed.
//
// A depth of 64 terms is in LDS twice, 128 KiB: while the matrix cores take one,
// buffer loads write the other straight into LDS. These loads check their
// range, so rows behind an operand's last are zero. LDS holds 16-byte chunks in an
// order that spreads the 256 bytes of a cycle (16 lanes by row, 32 by term) over all
// 64 banks:
//   by row   128 bytes a row, chunk c of row r at c ^ (r / 2 % 8)
//   by term  512 bytes a term, chunk c of term k at c ^ (4 (k % 4))
// The counters then show no conflict. With r % 8 and 2 (k % 4), two lanes to a bank,
// conflicts took a quarter of the cycles and 1 to 2 % of the time.
//
// float32 operands come as two f16 pieces, value = hi + lo, scaled to the f16
// range by a power of two; their product is hi lo + lo hi + hi hi, three runs over
// the same terms, the small ones first, while a sum's roundings are small too. What
// is left out is below 2^-22 of the factors.
#pragma once

#include "loss_params.h"
#include "mcpu_common.h"

namespace mcpu {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <typename T> __device__ __forceinline__ f32x16 mma32(s16x8 a, s16x8 b, f32x16 c) {
  if constexpr (std::is_same_v<T, bf16>)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                  0);
}

struct Operand {
  const void* base;   // first element of the first piece
  int64_t ld;         // elements between rows, or between terms
  int64_t piece;      // elements between the pieces
  int64_t span;       // elements from a piece's first to behind its last
};

struct ProductParams {
  Operand a, b;
  int64_t depth;   // terms, a multiple of 64
  int runs;        // 1, or 3 for operands of two pieces
};

constexpr int kTileBytes = kLossTile * kLossDepth * 2;

// Where an operand's tile of one depth begins, as a buffer that ends with the piece;
// behind the last depth (not `any`) an empty one, whose loads leave zeros.
template <bool TERM>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t tile_rsrc(const Operand& o, int64_t row0, int64_t k0, bool second,
                                                            bool any) {
  const int64_t at = TERM ? k0 * o.ld + row0 : row0 * o.ld + k0;
  const char* base = static_cast<const char*>(o.base) + 2 * (at + (second ? o.piece : 0));
  int64_t left = 2 * (o.span - at);
  left = left < 0 || !any ? 0 : left > 0xfffffff0ll ? 0xfffffff0ll : left;
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), 0, static_cast<int>(static_cast<uint32_t>(left)),
                                           0x00020000);
}

// This wave's eighth of a tile, four loads of 1 KiB.
template <bool TERM>
__device__ __forceinline__ void tile_load(char* lds, __amdgpu_buffer_rsrc_t r, uint32_t ld2, int wave, int lane) {
  using lds_ptr = __attribute__((address_space(3))) void*;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int piece = wave * 4 + i;
    uint32_t off;
    if constexpr (TERM) {
      const int k = piece * 2 + (lane >> 5);
      off = k * ld2 + (((lane & 31) ^ (4 * (k & 3))) << 4);
    } else {
      const int r = piece * 8 + (lane >> 3);
      off = r * ld2 + (((lane & 7) ^ (r >> 1 & 7)) << 4);
    }
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr)(lds + piece * 1024), 16, off, 0, 0, 0);
  }
}

// A lane's eight terms 16 ks + 8 (lane / 32) + 0..7 of row r0 + lane % 32.
template <bool TERM> __device__ __forceinline__ s16x8 tile_frag(const char* lds, int r0, int ks, int lane) {
  if constexpr (TERM) {
    using tr_ptr = s16x4 __attribute__((address_space(3)))*;
    const int kk = (lane & 15) >> 2;
    const int k = ks * 16 + 8 * (lane >> 5) + kk;
    const int col = r0 + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
    const char* at = lds + k * 512 + (((col >> 3) ^ (4 * kk)) << 4) + ((col & 4) << 1);
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)at);
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)(at + 4 * 512));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  } else {
    const int r = r0 + (lane & 31);
    return *reinterpret_cast<const s16x8*>(lds + r * 128 + (((ks * 2 + (lane >> 5)) ^ (r >> 1 & 7)) << 4));
  }
}

// Accumulators of a wave: v[j][i][e] is D at
//   m = m0 + 128 (wave / 4) + 32 i + 8 (e / 4) + 4 (lane / 32) + e % 4
//   n = n0 + 64 (wave % 4) + 32 j + lane % 32.
struct Acc {
  f32x16 v[2][4];
};

// A workgroup's LDS: both operands' tiles, twice. Four arrays, not one, for the
// compiler to see that what is read is not what the loads on their way write.
#define MCPU_TILE_LDS(a0, b0, a1, b1)                              \
  __shared__ __attribute__((aligned(1024))) char a0[kTileBytes]; \
  __shared__ __attribute__((aligned(1024))) char b0[kTileBytes]; \
  __shared__ __attribute__((aligned(1024))) char a1[kTileBytes]; \
  __shared__ __attribute__((aligned(1024))) char b1[kTileBytes]

// Depths [kt0, kt1) of the tile at (m0, n0), counted over all runs.
template <typename T, bool TA, bool TB>
__device__ __forceinline__ void tile_product(const ProductParams& p, int64_t m0, int64_t n0, int kt0, int kt1, char* a0,
                                             char* b0, char* a1, char* b1, Acc& acc) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = (wave >> 2) * 128, wn = (wave & 3) * 64;
  const int depths = static_cast<int>(p.depth / kLossDepth);
  const uint32_t lda2 = static_cast<uint32_t>(p.a.ld * 2), ldb2 = static_cast<uint32_t>(p.b.ld * 2);
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc.v[j][i][e] = 0.f;
  if (kt0 >= kt1) return;

  auto load = [&](char* la, char* lb, int kt) {
    const int run = kt >= 2 * depths ? 2 : kt >= depths ? 1 : 0;
    const int64_t k0 = int64_t{kt - run * depths} * kLossDepth;
    tile_load<TA>(la, tile_rsrc<TA>(p.a, m0, k0, p.runs > 1 && run == 1, kt < kt1), lda2, wave, lane);
    tile_load<TB>(lb, tile_rsrc<TB>(p.b, n0, k0, p.runs > 1 && run == 0, kt < kt1), ldb2, wave, lane);
  };
  auto step = [&](const char* la, const char* lb, char* na, char* nb, int kt) {
    // This wave's loads have arrived, then every wave's; and no wave reads the other buffer any more.
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    // A wave that multiplies goes before one that still sends its loads (1 to 2 %).
    __builtin_amdgcn_s_setprio(0);
    load(na, nb, kt + 1);
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(1);
    // Operands of the next 16 terms are read while these multiply, a read beside
    // each matrix instruction: 4 % faster than a read of all before their use.
    s16x8 a[2][4], b[2][2];
    auto frags = [&](int to, int ks) {
#pragma unroll
      for (int j = 0; j < 2; ++j) b[to][j] = tile_frag<TB>(lb, wn + 32 * j, ks, lane);
#pragma unroll
      for (int i = 0; i < 4; ++i) a[to][i] = tile_frag<TA>(la, wm + 32 * i, ks, lane);
    };
    frags(0, 0);
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      if (ks < 3) frags((ks + 1) & 1, ks + 1);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc.v[j][i] = mma32<T>(a[ks & 1][i], b[ks & 1][j], acc.v[j][i]);
    }
    constexpr int kReads = 2 * (TB ? 2 : 1) + 4 * (TA ? 2 : 1);
    __builtin_amdgcn_sched_group_barrier(0x100, kReads, 0);
#pragma unroll
    for (int u = 0; u < 32; ++u) {
      __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
      if (u % 8 < 6 && u < 24) __builtin_amdgcn_sched_group_barrier(0x100, kReads / 6, 0);
    }
  };
  load(a0, b0, kt0);
  int kt = kt0;
  for (; kt + 2 <= kt1; kt += 2) {
    step(a0, b0, a1, b1, kt);
    step(a1, b1, a0, b0, kt + 1);
  }
  if (kt < kt1) step(a0, b0, a1, b1, kt);
  // Nothing is on its way into LDS when the workgroup ends.
  __builtin_amdgcn_s_waitcnt(0x0070);
}

// The tile a workgroup takes, of `mt` x `nt` tiles: the workgroups of one XCD
// (every eighth) take neighbours, eight along m, then the next n.
__device__ __forceinline__ bool tile_of(int64_t id, int64_t mt, int64_t nt, int64_t& m, int64_t& n) {
  const int64_t all = mt * nt;
  if (id >= all) return false;
  const int64_t x = id & 7, per = all >> 3, more = all & 7;
  const int64_t at = x * per + (x < more ? x : more) + (id >> 3);
  const int64_t group = at / (8 * nt), in = at - group * 8 * nt;
  const int64_t high = mt - group * 8 < 8 ? mt - group * 8 : 8;
  n = in / high;
  m = group * 8 + in - n * high;
  return true;
}

}  // namespace mcpu
