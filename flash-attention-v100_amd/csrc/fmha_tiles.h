// What the kernels of this directory share: types, MFMA wrappers, the swizzled 64-row LDS tile with its copies and reads for both
// MFMA shapes, staging tiles for output rows, waits.  Included inside each translation unit, so that each has its own.
#ifndef FMHA_TILES_H_
#define FMHA_TILES_H_

#include <hip/hip_runtime.h>
#include <stdint.h>
#include <math.h>
#include <type_traits>
#include <utility>

#include "block_map.h"

namespace {

typedef _Float16 half_t;
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef float f4v __attribute__((ext_vector_type(4)));

constexpr int kResident = 32;      // resident positions per wave
constexpr int kTile = 64;          // streamed rows per LDS tile
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

template <int D>
struct TileGeom {
  static constexpr int kKSteps = D / 16;                   // MFMA k-steps over D
  static constexpr int kDBlocks = D / 32;                  // 32-row blocks over D
};

__device__ __forceinline__ f16v mfma(h8 a, h8 b, f16v c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f4v mfma16(h8 a, h8 b, f4v c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// dS for two neighbouring positions: fp16(-p.lo * x0) and fp16(-p.hi * x1), the products in fp32, as
// two mixed-precision FMAs that read the fp16 halves of p directly (the same bits as converting p to
// fp32, multiplying and converting back, in 2 instructions instead of 5).
typedef unsigned u4v __attribute__((ext_vector_type(4)));
__device__ __forceinline__ unsigned neg_mul_to_f16x2(unsigned p_pair, float x0, float x1) {
  unsigned r;
  asm("v_fma_mixlo_f16 %0, %1, -%2, 0 op_sel_hi:[1,0,0]\n\t"
      "v_fma_mixhi_f16 %0, %1, -%3, 0 op_sel:[1,0,0] op_sel_hi:[1,0,0]"
      : "=&v"(r)
      : "v"(p_pair), "v"(x0), "v"(x1));
  return r;
}
// y[.] = fp16(-p[.] * x[.]) for the 8 values of one B-operand fragment
__device__ __forceinline__ h8 neg_mul_to_f16x8(h8 p, const float* x) {
  const u4v pp = __builtin_bit_cast(u4v, p);
  u4v r;
#pragma unroll
  for (int j = 0; j < 4; ++j) r[j] = neg_mul_to_f16x2(pp[j], x[2 * j], x[2 * j + 1]);
  return __builtin_bit_cast(h8, r);
}

// Element strides of a (batch, n, head, d) tensor whose last dimension is
// contiguous.  The dense layout of reference kernel/fused_mha_kernel.cu:57-59 is
// {n*head*d, head*d, d}.
struct Strides {
  long b;
  int n, h;
};

// Combine a value with the one held by the lane 32 positions away.
__device__ __forceinline__ float other_half(float x) {
  int xi = __float_as_int(x);
  auto r = __builtin_amdgcn_permlane32_swap(xi, xi, false, false);
  // r[0]: lanes 0-31 keep own, lanes 32-63 get lane-32's; r[1] the converse.
  int mine_or_other = (threadIdx.x & 32) ? r[0] : r[1];
  return __int_as_float(mine_or_other);
}

// Streamed-row index of accumulator register r in row-block rb for half hh.
__device__ __forceinline__ int acc_row(int rb, int r, int hh) {
  return rb * 32 + 8 * (r >> 2) + 4 * hh + (r & 3);
}

// The rows of a staging tile as they leave.  All of them are asked for before the first is stored, and only a block with rows
// past the end looks at each: one after the other, as read, wait, test and store, they take 200 cycles each.
// Kernels in graphs of 20 calls, us one after the other and as it is, forward, then backward, N x slices: D = 64 77 x 8 causal
// 5.76, 5.67 and 6.86, 6.61; 128 x 4 5.15, 5.06 and 6.48, 6.31; 1024 x 64 causal 17.3, 17.2 and 43.4, 43.1; D = 128 200 x 48
// causal 9.45, 9.32 and 14.8 both; 2048 x 80 causal 95.7, 95.4 and 296, 295.
template <int D, int kPitch, typename Piece>
__device__ __forceinline__ void store_staged(half_t* __restrict__ base, int row_stride, int row0, int n, int lane,
                                             const char* __restrict__ stage, int upper_off) {
  constexpr int kLanesPerRow = D / 8, kRowsPerPass = 64 / kLanesPerRow, kPasses = kResident / kRowsPerPass;
  const int r_in = lane / kLanesPerRow, ch = lane % kLanesPerRow;
  union Row {
    Piece piece[16 / sizeof(Piece)];
    h8 v;
  } rows[kPasses];
#pragma unroll
  for (int pass = 0; pass < kPasses; ++pass) {
    const int r = pass * kRowsPerPass + r_in;
    const char* const src = stage + (r & 15) * kPitch + (r >> 4) * upper_off + ch * 16;
#pragma unroll
    for (int e = 0; e < (int)(16 / sizeof(Piece)); ++e) rows[pass].piece[e] = *reinterpret_cast<const Piece*>(src + e * sizeof(Piece));
  }
  char* const out = reinterpret_cast<char*>(base + (long)row0 * row_stride);
  const unsigned off = r_in * row_stride * 2 + ch * 16;
  auto store = [&](int pass) __attribute__((always_inline)) {
    *reinterpret_cast<h8*>(out + (long)pass * kRowsPerPass * 2 * row_stride + off) = rows[pass].v;
  };
  if (row0 + kResident <= n) {
#pragma unroll
    for (int pass = 0; pass < kPasses; ++pass) store(pass);
  } else {
#pragma unroll
    for (int pass = 0; pass < kPasses; ++pass)
      if (row0 + pass * kRowsPerPass + r_in < n) store(pass);
  }
}

// Store a [D][32 resident] fp32 accumulator, scaled, as fp16 rows of a dense
// (B, N, H, D) tensor, through a staging tile in LDS that belongs to the wave
// (32 rows of kStagePitch bytes): each lane first writes the 4-feature pieces it
// holds of its own row, then the wave reads the tile back row-wise, so that
// every row leaves as whole 16-byte pieces written by neighbouring lanes (a
// 256-byte row by 16 lanes, as the reference's epilogue does with its 128-bit
// stores, kernel/fused_mha_kernel.cu:318-322, 714-734).  Lane (i, hh) owns row
// row0 + i; per 32-feature block it holds features 8*g + 4*hh + 0..3 for g = 0..3.
// The caller makes sure (with a block barrier) that nobody still reads what the
// staging tile overwrites.
template <int D>
struct StageGeom {
  // bytes per row: a row plus 8, so that the lanes of a half wave, which write 8 bytes each to
  // 32 different rows, spread over the banks; the rows are read back as 8-byte pieces.
  // (Measured: no bank conflicts with D = 64; with D = 128 four conflict cycles per 8-byte
  // store instruction remain whatever the padding or swizzle, 64 cycles per wave and launch.)
  static constexpr int kPitch = D * 2 + 8;
  static constexpr int kBytes = kResident * kPitch;  // per wave
};
template <int D>
__device__ __forceinline__ void store_resident(half_t* __restrict__ base, int row_stride, int row0, int n,
                                               const f16v (&acc)[TileGeom<D>::kDBlocks], float mul, int lane,
                                               char* __restrict__ stage, int my_row = -1,
                                               int upper_off = 16 * StageGeom<D>::kPitch) {
  // my_row: the row (0..31, relative to row0) this lane's column of the accumulator belongs
  // to, when that is not lane & 31; upper_off: where rows 16..31 are staged, relative to `stage`,
  // when the staging tile is not contiguous (see fmha_bwd_dq_spill_kernel for both)
  constexpr int kPitch = StageGeom<D>::kPitch;
  const int i = my_row < 0 ? (lane & 31) : my_row, hh = lane >> 5;
  char* mine = stage + (i & 15) * kPitch + (i >> 4) * upper_off + hh * 8;
#pragma unroll
  for (int db = 0; db < TileGeom<D>::kDBlocks; ++db) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      h4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = (half_t)(acc[db][4 * g + e] * mul);
      *reinterpret_cast<h4*>(mine + (db * 32 + 8 * g) * 2) = v;
    }
  }
  __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): the wave's own writes have landed
  asm volatile("" ::: "memory");
  store_staged<D, kPitch, h4>(base, row_stride, row0, n, lane, stage, upper_off);
}

// Blocks of a persistent work group (schedule: block_map.h).
struct PersistentBlocks {
  int total;
  __device__ __forceinline__ int lin(int r) const {  // >= total: this group has no block in round r
    return fmha_persistent_block(r, blockIdx.x, gridDim.x);
  }
  __device__ __forceinline__ int next_round(int r) const {  // the next round with a block for this group, or -1
    return fmha_persistent_next_round(r, blockIdx.x, gridDim.x, total);
  }
};

// ---------------------------------------------------------------------------
// 64-row tiles copied global -> LDS by global_load_lds_dwordx4 (no registers in
// between).  One wave-level instruction moves 1 KiB: 16 rows x 64 bytes, every
// 4 lanes reading one 64-byte row segment.  The tile is an array of such 1 KiB
// blocks, block (R, C) = rows 16R..16R+15, bytes 64C..64C+63 of each row.
// Inside a block the 16-byte chunk c4 of row r16 sits at
//     r16 * 64 + ((c4 ^ swz(r16 >> 2)) * 16),
// which makes all read patterns below bank-conflict free without padding:
//   rows:  16 lanes read the same chunk of 16 rows      (128-bit reads)
//   cols:  16 lanes read 4 rows x 32 bytes, transposed  (ds_read_b64_tr_b16)
// ---------------------------------------------------------------------------
__host__ __device__ constexpr int swz(int rows4) { return -rows4 & 3; }
template <int D>
struct SwzTile {
  static constexpr int kNC = D / 32;              // 64-byte column groups per row
  static constexpr int kBytes = kTile * D * 2;
  static constexpr int kInstrs = 4 * kNC;         // 1 KiB copies per tile
  __host__ __device__ static constexpr int block_off(int R, int C) { return (R * kNC + C) * 1024; }
};

// Per-lane source of copy instruction t (block R = t / kNC, C = t % kNC):
// byte offset from the tile's first row, and the row inside the tile.
template <int D>
__device__ __forceinline__ void copy_src(int t, int lane, int row_stride, int& row, int& goff) {
  const int R = t / SwzTile<D>::kNC, C = t % SwzTile<D>::kNC;
  const int r16 = lane >> 2, pos = lane & 3;
  const int c4 = pos ^ swz(r16 >> 2);
  row = 16 * R + r16;
  goff = (row * row_stride + (4 * C + c4) * 8) * 2;  // bytes
}

// One 1 KiB copy: lane l fetches 16 bytes at tile_base + voff and they land in
// LDS at lds_block + 16 * l.  Written as inline asm on purpose: the compiler's
// wait-count insertion then knows nothing of the copy, so it cannot make later
// LDS reads wait for it (it cannot tell the ring slots apart and would wait for
// every copy in flight); the waits for these copies are the explicit wait_vm<>
// calls in the kernels.  tile_base and lds_block must be wave-uniform.
// The LDS address travels in m0, which the compiler reserves for itself and
// does not accept as a clobber: the statement saves and restores it, so a value
// the compiler keeps there (indirect register indexing, its own LDS copies)
// survives.
__device__ __forceinline__ void copy16(const half_t* tile_base, int voff, char* lds_block) {
  const unsigned lds_addr = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)lds_block;
  unsigned saved_m0;
  asm volatile(
      "s_mov_b32 %0, m0\n\t"
      "s_mov_b32 m0, %3\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %1, %2\n\t"
      "s_mov_b32 m0, %0"
      : "=&s"(saved_m0)
      : "v"(voff), "s"(tile_base), "s"(lds_addr)
      : "memory");
}
// The same for dS.  STREAM: with the hint that it is read once, which keeps it from displacing the tiles other work groups
// re-read out of the L2.  SHARED: other work groups of the launch have written it (sc1: not out of this XCD's L2, see store_ds).
template <bool SHARED, bool STREAM>
__device__ __forceinline__ void copy16_ds(const half_t* tile_base, int voff, char* lds_block) {
  const unsigned lds_addr = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)lds_block;
  unsigned saved_m0;
#define FMHA_COPY16(HINTS)                            \
  asm volatile(                                       \
      "s_mov_b32 %0, m0\n\t"                          \
      "s_mov_b32 m0, %3\n\t"                          \
      "s_nop 0\n\t"                                   \
      "global_load_lds_dwordx4 %1, %2" HINTS "\n\t"   \
      "s_mov_b32 m0, %0"                              \
      : "=&s"(saved_m0)                               \
      : "v"(voff), "s"(tile_base), "s"(lds_addr)      \
      : "memory")
  if constexpr (SHARED && STREAM) FMHA_COPY16(" sc1 nt");
  else if constexpr (SHARED) FMHA_COPY16(" sc1");
  else if constexpr (STREAM) FMHA_COPY16(" nt");
  else FMHA_COPY16("");
#undef FMHA_COPY16
}

// kCount copies of 1 KiB to consecutive blocks of LDS: lane l's 16 bytes of block u land at lds + 1024 * u + 16 * l.
// The instruction's offset counts for both addresses, so they come from base + voff + 64 * u with voff lowered by
// 960 * u.
template <int kCount>
__device__ __forceinline__ void copy16_blocks(const half_t* base, int voff, unsigned lds) {
  static_assert(kCount == 2 || kCount == 4, "");
  unsigned saved_m0;
  if constexpr (kCount == 2) {
    asm volatile(
        "s_mov_b32 %0, m0\n\t"
        "s_mov_b32 m0, %2\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %3, %1\n\t"
        "global_load_lds_dwordx4 %4, %1 offset:1024\n\t"
        "s_mov_b32 m0, %0"
        : "=&s"(saved_m0)
        : "s"(base), "s"(lds), "v"(voff), "v"(voff - 960)
        : "memory");
  } else {
    asm volatile(
        "s_mov_b32 %0, m0\n\t"
        "s_mov_b32 m0, %2\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %3, %1\n\t"
        "global_load_lds_dwordx4 %4, %1 offset:1024\n\t"
        "global_load_lds_dwordx4 %5, %1 offset:2048\n\t"
        "global_load_lds_dwordx4 %6, %1 offset:3072\n\t"
        "s_mov_b32 m0, %0"
        : "=&s"(saved_m0)
        : "s"(base), "s"(lds), "v"(voff), "v"(voff - 960), "v"(voff - 1920), "v"(voff - 2880)
        : "memory");
  }
}

// The same with 4 bytes per lane (256 bytes per instruction): lane l fetches the
// dword at base + voff and it lands in LDS at lds_dst + 4 * l.
__device__ __forceinline__ void copy4(const float* base, int voff, char* lds_dst) {
  const unsigned lds_addr = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)lds_dst;
  unsigned saved_m0;
  asm volatile(
      "s_mov_b32 %0, m0\n\t"
      "s_mov_b32 m0, %3\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dword %1, %2\n\t"
      "s_mov_b32 m0, %0"
      : "=&s"(saved_m0)
      : "v"(voff), "s"(base), "s"(lds_addr)
      : "memory");
}

// rows pattern: lane (i, hh) reads chunk 2*kk + hh of row rb*32 + i.
// Two lane offsets (kk even / odd); the rest is an immediate.
template <int D>
__device__ __forceinline__ void swz_rows_off(int lane, int (&off)[2]) {
  const int i = lane & 31, hh = lane >> 5, r16 = i & 15, g = swz(r16 >> 2);
  const int base = (i >> 4) * SwzTile<D>::kNC * 1024 + r16 * 64;
  off[0] = base + ((hh ^ g) * 16);
  off[1] = base + (((2 + hh) ^ g) * 16);
}
template <int D>
__device__ __forceinline__ h8 swz_rows(const char* tile, int rb, int kk, const int (&off)[2]) {
  return *reinterpret_cast<const h8*>(tile + off[kk & 1] + SwzTile<D>::block_off(2 * rb, kk >> 1));
}
// cols pattern: MFMA A operand, rows = features db*32 + (lane & 31), k = streamed
// rows of chunk c16 in accumulator order.  Two lane offsets (rows +0 / +8).
template <int D>
__device__ __forceinline__ void swz_cols_off(int lane, int (&off)[2]) {
  const int L = lane & 15, half = (lane >> 4) & 1, hh = lane >> 5;
  const int c4 = 2 * half + ((L & 3) >> 1);
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int r16 = 8 * e + 4 * hh + (L >> 2);
    off[e] = r16 * 64 + ((c4 ^ swz(r16 >> 2)) * 16) + (L & 1) * 8;
  }
}
template <int D>
__device__ __forceinline__ h8 swz_cols(const char* tile, int c16, int db, const int (&off)[2]) {
  typedef __attribute__((address_space(3))) s4 lds_s4;
  const char* p = tile + SwzTile<D>::block_off(c16, db);
  s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(p + off[0]));
  s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(p + off[1]));
  return __builtin_bit_cast(h8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

// The same reads through LDS addresses formed by the caller (tile + off[e]) and hidden from the optimiser:
// seen whole, it may split tile + off[e] + constant into a loop-invariant part per fragment, kept in a
// register each (and spilled), and the ring slot; opaque, the constant is the instruction's immediate offset.
__device__ __forceinline__ unsigned opaque_lds_address(const char* p) {
  unsigned a = (unsigned)(uintptr_t)(__attribute__((address_space(3))) const char*)p;
  asm volatile("" : "+v"(a));
  return a;
}
template <int D>
__device__ __forceinline__ h8 swz_rows_at(unsigned a_even, unsigned a_odd, int rb, int kk) {
  typedef __attribute__((address_space(3))) h8 lds_h8;
  return *(const lds_h8*)(uintptr_t)(((kk & 1) ? a_odd : a_even) + (unsigned)SwzTile<D>::block_off(2 * rb, kk >> 1));
}
template <int D>
__device__ __forceinline__ h8 swz_cols_at(unsigned a0, unsigned a1, int c16, int db) {
  typedef __attribute__((address_space(3))) s4 lds_s4;
  const unsigned o = SwzTile<D>::block_off(c16, db);
  s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(uintptr_t)(a0 + o));
  s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(uintptr_t)(a1 + o));
  return __builtin_bit_cast(h8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

// ---------------------------------------------------------------------------
// 16 x 16 x 32 MFMAs over the same tiles.  At the power cap they do 13 % more products per second than the 32 x 32 x 16
// ones (registers only, random operands, all CUs busy: 1,766 against 1,555 TFLOP/s; with each A operand read from LDS for
// 2 x 16 columns 1,580 against 1,400), so the kernels that run there use them.  They are twice as many instructions, which
// a wave alone on its SIMD feels (B1 H2 N4000 forward: 51 -> 59 us), and where vector instructions are the bound they gain
// nothing (B1 H12 N8192 D64 forward: 218 -> 223 us): those kernels keep the others.
//
// Both give the same bits.  One 16 x 16 x 32 MFMA adds the products of its lanes 0..31 first, then those of lanes
// 32..63, each the way a 32 x 32 x 16 MFMA adds its 16; and the streamed rows are dealt out so that these are the same 16:
// of 32 streamed rows kc, row block p (0 or 1) has, in MFMA row 4 g + r (held by lanes 16 g .. in register r), the row
//     32 kc + 16 (g >> 1) + 8 p + 4 (g & 1) + r.
// The second GEMM takes rows 32 kc .. as one step, register e = 4 p + r of lane group g as its k = 8 g + e.
// ---------------------------------------------------------------------------
template <int D>
struct Geom16 {
  static constexpr int kKS = D / 32;  // steps over the features
  static constexpr int kDB = D / 16;  // blocks of 16 features
};
// first of the four streamed rows, inside 32, that lane group g holds in row block p
__device__ __forceinline__ int acc16_row(int p, int g) { return 16 * (g >> 1) + 8 * p + 4 * (g & 1); }
// rows pattern: lane (m, g) reads chunk g of the row of MFMA row m; two lane offsets (row block even / odd).
template <int D>
__device__ __forceinline__ int rows16_off(int lane, int p) {
  const int m = lane & 15, g = lane >> 4, r16 = 8 * p + (m & 7);
  return (m >> 3) * SwzTile<D>::kNC * 1024 + r16 * 64 + ((g ^ swz(r16 >> 2)) * 16);
}
template <int D>
__device__ __forceinline__ h8 rows16_at(unsigned a_even, unsigned a_odd, int rb, int kk) {
  typedef __attribute__((address_space(3))) h8 lds_h8;
  return *(const lds_h8*)(uintptr_t)(((rb & 1) ? a_odd : a_even) + (unsigned)SwzTile<D>::block_off(rb & 2, kk));
}
// cols pattern: MFMA A operand, rows = features 16 db + (lane & 15), k = 32 streamed rows kc in accumulator order.  Two
// lane offsets (rows +0 / +8) for even db; odd ones are 32 bytes away, one way or the other.
template <int D>
__device__ __forceinline__ int cols16_off(int lane, int p, int odd) {
  const int L = lane & 15, g = lane >> 4, r16 = 8 * p + 4 * (g & 1) + (L >> 2);
  return (g >> 1) * SwzTile<D>::kNC * 1024 + r16 * 64 + (((2 * odd + ((L & 3) >> 1)) ^ swz(r16 >> 2)) * 16) + (L & 1) * 8;
}
template <int D>
struct Cols16 {
  unsigned a[2][2];  // [rows +0 / +8][feature block even / odd]
  __device__ __forceinline__ Cols16(const char* tile, int lane) {
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int odd = 0; odd < 2; ++odd) a[p][odd] = opaque_lds_address(tile + cols16_off<D>(lane, p, odd));
  }
  __device__ __forceinline__ h8 at(unsigned slot, int kc, int db) const {
    typedef __attribute__((address_space(3))) s4 lds_s4;
    const unsigned o = slot + SwzTile<D>::block_off(2 * kc, db >> 1);
    s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(uintptr_t)(a[0][db & 1] + o));
    s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(uintptr_t)(a[1][db & 1] + o));
    return __builtin_bit_cast(h8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  }
};
// s_waitcnt vmcnt(N) with the other counters left alone.  Issued through the
// builtin (not inline asm) so that the compiler's wait-count bookkeeping sees it.
template <int N>
__device__ __forceinline__ void wait_vm() {
  static_assert(N >= 0 && N < 64, "vmcnt immediate");  // bits 3:0 and 15:14 of the immediate
  __builtin_amdgcn_s_waitcnt(0x0F70 | (N & 15) | ((N >> 4) << 14));
}

// A wave's 32 resident rows on their way to registers: copied to D / 16 KiB of LDS that are the wave's own (rows row0 .. of a
// slice, row N-1 in the place of those past the end) and, once they are there, read as MFMA B operands.  Loaded straight to
// registers, neighbouring lanes ask for 16 bytes of different rows each, and the CU's path to memory takes 64 cycles for
// what a copy takes 16 for, 64 bytes of a row from every four lanes: 2,000 to 4,000 cycles at the start of a block.
// Kernels in graphs of 20 calls, us loaded straight and this way, forward and backward, N x slices: D = 64 128 x 4 4.92, 4.70 and 6.31,
// 5.87; 300 x 80 causal 7.38, 7.21 and 13.3, 12.4; 1024 x 64 causal 16.7, 16.6 and 43.1, 42.1; D = 128 128 x 32 6.69, 6.13 and 9.86,
// 8.59; 200 x 48 causal 9.08, 8.79 and 14.9, 13.6; 700 x 24 13.9, 13.5 and 34.1, 33.2; 2048 x 80 causal 94.6, 93.3 and 296, 295.
template <int D>
__device__ __forceinline__ void copy_rows(const half_t* slice, int stride, int row0, int n, int lane, char* lds) {
  constexpr int kNC = SwzTile<D>::kNC, kBack = 960 * (kNC - 1);  // see copy16_blocks
  row0 = min(row0, n - 1);
  const half_t* const base = slice + (long)row0 * stride - kBack / 2;
  const unsigned to = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
  const int r16 = lane >> 2, col = ((lane & 3) ^ swz(lane >> 4)) * 16 + kBack;
#pragma unroll
  for (int R = 0; R < 2; ++R) {
    const int row = min(16 * R + r16, n - 1 - row0);
    copy16_blocks<kNC>(base, row * stride * 2 + col, to + SwzTile<D>::block_off(R, 0));
  }
}
template <int D>
struct StagedRows {
  const char* at;
  int lane;
  __device__ __forceinline__ h8 wide(int kk) const {  // for 32 x 32 MFMAs: features 16 kk .. of row lane & 31
    int off[2];
    swz_rows_off<D>(lane, off);
    return swz_rows<D>(at, 0, kk, off);
  }
  __device__ __forceinline__ h8 narrow(int kk, int cb) const {  // for 16 x 16 ones: features 32 kk .. of row 16 cb + (lane & 15)
    const int i = lane & 15;
    return *reinterpret_cast<const h8*>(at + SwzTile<D>::block_off(cb, kk) + i * 64 + (((lane >> 4) ^ swz(i >> 2)) * 16));
  }
};
// The copies are there: read them.
__device__ __forceinline__ void staged_rows_landed() {
  wait_vm<0>();
  asm volatile("" ::: "memory");
}
// They are read: others may take their place.
__device__ __forceinline__ void staged_rows_read() {
  __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
  asm volatile("" ::: "memory");
}

// Over the four lanes with the same l & 15: first the two that are 32 apart, then the others.
__device__ __forceinline__ float max_over_groups(float x) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_int(x), __float_as_int(x), false, false);
  x = fmaxf(__int_as_float(r[0]), __int_as_float(r[1]));
  r = __builtin_amdgcn_permlane16_swap(__float_as_int(x), __float_as_int(x), false, false);
  return fmaxf(__int_as_float(r[0]), __int_as_float(r[1]));
}
// store_resident for accumulators of 16 x 16 blocks: acc[db][cb] has features 16 db + 4 g + 0..3 of resident position
// 16 cb + (lane & 15), to be scaled by mul[cb].
template <int D>
struct Stage16 {
  // bytes per row: the 8-byte pieces that 32 lanes write, 16 rows x 2, fall on different banks
  static constexpr int kPitch = D * 2 + 16;
  static constexpr int kBytes = kResident * kPitch;  // per wave
};
template <int D>
__device__ __forceinline__ void store_resident16(half_t* __restrict__ base, int row_stride, int row0, int n,
                                                 const f4v (*acc)[2], const float (&mul)[2], int lane,
                                                 char* __restrict__ stage, int row_of_0 = -1, int row_of_1 = -1,
                                                 int upper_off = 16 * Stage16<D>::kPitch) {
  // row_of_cb: the row (0..31, relative to row0) of this lane's column of block cb, when that is not 16 cb + (lane & 15);
  // upper_off: where rows 16..31 are staged, relative to `stage`, when the staging tile is not contiguous
  constexpr int kPitch = Stage16<D>::kPitch;
#pragma unroll
  for (int cb = 0; cb < 2; ++cb) {
    const int row = row_of_0 < 0 ? 16 * cb + (lane & 15) : cb ? row_of_1 : row_of_0;
    char* mine = stage + (row & 15) * kPitch + (row >> 4) * upper_off + (lane >> 4) * 8;
#pragma unroll
    for (int db = 0; db < D / 16; ++db) {
      h4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = (half_t)(acc[db][cb][e] * mul[cb]);
      *reinterpret_cast<h4*>(mine + db * 32) = v;
    }
  }
  __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): the wave's own writes have landed
  asm volatile("" ::: "memory");
  store_staged<D, kPitch, h8>(base, row_stride, row0, n, lane, stage, upper_off);
}

// Arguments of a kernel, asked for here: left to the compiler they come in four or five groups, each where it is first needed and
// each waited for by itself.  128-query forward, which also tests for a negative scale now instead of negating and
// choosing, us before and after, N x slices: D = 64 77 x 8 causal 5.66, 5.45; 512 x 192 21.8, 21.1; 1024 x 64 causal 17.2, 16.7; D =
// 128 200 x 48 causal 9.33, 9.08.  The kernels of the backward gain nothing from it.
__device__ __forceinline__ void load_now(const Strides& s) { asm volatile("" ::"s"(s.b), "s"(s.n), "s"(s.h)); }
__device__ __forceinline__ void load_now(const FmhaDivisor& v) { asm volatile("" ::"s"(v.d), "s"(v.mul), "s"(v.shift)); }
template <typename T>
__device__ __forceinline__ void load_now(T v) { asm volatile("" ::"s"(v)); }
template <typename... T>
__device__ __forceinline__ void load_all_now(const T&... v) { (load_now(v), ...); }

// Wait until at most n (0 to 4) of this wave's LDS reads are on their way.
__device__ __forceinline__ void wait_lds(int n) {
  if (n == 0) __builtin_amdgcn_s_waitcnt(0xC07F);
  else if (n == 1) __builtin_amdgcn_s_waitcnt(0xC17F);
  else if (n == 2) __builtin_amdgcn_s_waitcnt(0xC27F);
  else if (n == 3) __builtin_amdgcn_s_waitcnt(0xC37F);
  else __builtin_amdgcn_s_waitcnt(0xC47F);
}
// The same at this place in the program, so that the compiler adds no wait of its own in front of it.
__device__ __forceinline__ void wait_lds_pinned(int n) {
  __builtin_amdgcn_sched_barrier(0);
  wait_lds(n);
  __builtin_amdgcn_sched_barrier(0);
}
__device__ __forceinline__ void block_barrier() {
  __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): this wave's LDS reads have landed
  asm volatile("" ::: "memory");       // keep LDS accesses on their side of the barrier
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
// Wait until at most min(later, kMax) * kPer of this wave's copies are in flight.
template <int kPer, int kMax>
__device__ __forceinline__ void wait_vm_tiles(int later) {
  if constexpr (kMax == 0) {
    wait_vm<0>();
  } else {
    if (later >= kMax) wait_vm<kMax * kPer>();
    else wait_vm_tiles<kPer, kMax - 1>(later);
  }
}
template <int V>
struct IntTag { static constexpr int value = V; };
// f(IntTag<0>{}), f(IntTag<1>{}), .. f(IntTag<kN - 1>{}): unrolled whatever the size of the body.
template <typename F, int... I>
__device__ __forceinline__ void static_for_each(std::integer_sequence<int, I...>, F&& f) {
  (f(IntTag<I>{}), ...);
}
template <int kN, typename F>
__device__ __forceinline__ void static_for(F&& f) {
  static_for_each(std::make_integer_sequence<int, kN>{}, f);
}

}  // namespace
#endif  // FMHA_TILES_H_
