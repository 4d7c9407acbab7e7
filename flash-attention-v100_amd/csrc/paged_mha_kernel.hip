// Attention over a cache of keys and values in pages, its writing and its reading, for gfx950.  C ABI: paged_mha.h.
//
// Layouts: the cache is (pages, page_size, kv_head, d) with strides; q, k, v and o are (tokens, heads, d) with strides.  The
// rows of a key head are its query heads' rows of all new tokens, token by token, so that they share the keys they read.

#include <hip/hip_runtime.h>
#include <stdint.h>
#include <math.h>
#include <algorithm>

#include "paged_mha.h"
#include "fmha_tiles.h"
#include "paged_plan.h"

namespace {

typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef __bf16 b4 __attribute__((ext_vector_type(4)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));
typedef unsigned u2v __attribute__((ext_vector_type(2)));

// Bytes, not elements: slot and head fit 32 bits.
struct CacheStrides {
  long page;
  int slot, head;
};

struct PagedArgs {
  const char *q, *k, *v;
  const unsigned char *k_scale, *v_scale;
  char* o;
  const int *table, *keys, *ends;  // ends: cu_seqlens + 1, or null
  float* part_o;                   // of part p: rows_of_block x D sums, relative to the maximum
  float2* part_ml;                 // of part p: maximum (of exponents of 2) and sum of each row
  CacheStrides ks, vs, kss, vss;
  long q_batch, q_seq, q_head, table_stride;  // of q in bytes
  int batch, new_tokens, tokens;              // new_tokens: of each sequence, where ends is null; tokens: in all
  int head, kv_head, pages, width;
  FmhaDivisor group, page_size;  // group: query heads of a key head
  float c;                       // scale * log2(e)
  int causal, zero_rest;
  int target, least;  // parts aimed at and their least tiles; target 0: an item is a part
  int slots;          // parts there is room for: enough unless entries of ends go back
};

struct Sequence {
  int first, n;  // its tokens
  int keys;
  bool past;     // it has more keys than the page table has places
};
__device__ __forceinline__ Sequence sequence(const PagedArgs& a, int b) {
  Sequence s;
  if (a.ends) {
    const int lo = a.ends[b - 1], hi = a.ends[b];
    s.first = min(max(lo, 0), a.tokens);
    s.n = min(max(hi, s.first), a.tokens) - s.first;
  } else {
    s.first = b * a.new_tokens;
    s.n = a.new_tokens;
  }
  const int keys = max(a.keys[b], 0);
  const long places = (long)a.width * (int)a.page_size;
  s.past = keys > places;
  s.keys = s.past ? (int)places : keys;
  return s;
}

// The sequence that token t belongs to, or another one where it belongs to none; 64 lanes look together.  Where ends do not
// grow it is any sequence.
__device__ __forceinline__ int sequence_of(const int* ends, int batch, int t, int lane) {
  int lo = 0, size = batch;
  while (size > 64) {
    const int step = (size + 63) >> 6, at = lo + (lane + 1) * step;
    const int n = __popcll(__builtin_amdgcn_ballot_w64(at <= lo + size && ends[min(at, batch) - 1] <= t));
    lo += n * step;
    size = min(step, size - n * step);
  }
  lo += __popcll(__builtin_amdgcn_ballot_w64(lane < size && ends[lo + min(lane, size - 1)] <= t));
  return min(lo, batch - 1);
}

__device__ __forceinline__ long sum_over_wave(long x) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) x += __shfl_xor(x, d);
  return x;
}
__device__ __forceinline__ int scan_over_wave(int x, int lane) {  // with its own
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int y = __shfl_up(x, d);
    if (lane >= d) x += y;
  }
  return x;
}

// Tiles of a part.
template <int ROWS>
__device__ __forceinline__ int tiles_of_part(const PagedArgs& a, int lane) {
  if (a.target == 0) return 1 << 30;
  long tiles = 0;
  for (int b = lane; b < a.batch; b += 64) {
    const Sequence s = sequence(a, b);
    tiles += (long)paged_blocks(s.n * a.group, ROWS) * paged_tiles(s.keys);
  }
  return paged_tiles_of_part(sum_over_wave(tiles) * a.kv_head, a.target, a.least);
}

// Part `w` of the launch, or b = -1; with parts of sequences before it counted in `before`.
struct Part {
  int b, head, block, p, parts, number;
  Sequence s;
};
template <int ROWS>
__device__ __forceinline__ Part part_of(const PagedArgs& a, int w, int lane) {
  const int per = tiles_of_part<ROWS>(a, lane);
  auto parts_of = [&](int b) __attribute__((always_inline)) {  // of one key head
    if (b >= a.batch) return 0;
    const Sequence s = sequence(a, b);
    return paged_blocks(s.n * a.group, ROWS) * paged_parts(paged_tiles(s.keys), per);
  };
  Part r;
  r.b = -1;
  int all = 0;
  for (int b0 = 0; b0 < a.batch; b0 += 64) all += __shfl(scan_over_wave(parts_of(b0 + lane), lane), 63);
  const int number = paged_spread(w, all * a.kv_head);
  if (number >= all * a.kv_head) return r;
  int before = 0;
  for (int b0 = 0; b0 < a.batch; b0 += 64) {
    const int mine = parts_of(b0 + lane), upto = before + scan_over_wave(mine, lane);
    const unsigned long long past = __builtin_amdgcn_ballot_w64(upto * a.kv_head > number);
    if (past) {
      const int l = __builtin_ctzll(past);
      const int b = b0 + l, of_head = __shfl(mine, l), base = (__shfl(upto, l) - of_head) * a.kv_head;
      r.b = __builtin_amdgcn_readfirstlane(b);
      r.s = sequence(a, r.b);
      if (a.target && number >= a.slots) {
        r.b = -1;
        return r;
      }
      r.parts = paged_parts(paged_tiles(r.s.keys), per);
      const int local = number - base;
      r.head = __builtin_amdgcn_readfirstlane(local / of_head);
      const int in_head = local - r.head * of_head;
      r.block = __builtin_amdgcn_readfirstlane(in_head / r.parts);
      r.p = __builtin_amdgcn_readfirstlane(in_head - r.block * r.parts);
      r.number = number;
      return r;
    }
    before = __shfl(upto, 63);
  }
  return r;
}

template <bool BF>
__device__ __forceinline__ f4v mma16(h8 x, h8 y, f4v z) {
  if constexpr (BF) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, x), __builtin_bit_cast(b8, y), z, 0, 0, 0);
  else return mfma16(x, y, z);
}
// Two values to the 16-bit type, to nearest.
template <bool BF>
__device__ __forceinline__ unsigned pack2(float x, float y) {
  if constexpr (BF) return __builtin_bit_cast(unsigned, b2{(__bf16)x, (__bf16)y});
  else return __builtin_bit_cast(unsigned, h2{(half_t)x, (half_t)y});
}
// Eight e4m3 values times 2^(byte - 127), which is exact (paged_mha.h): the instruction takes the exponent of its scale.
template <bool BF>
__device__ __forceinline__ u4v from_e4m3(unsigned lo, unsigned hi, float scale) {
  u4v r;
  if constexpr (BF) {
    r[0] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false));
    r[1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true));
    r[2] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false));
    r[3] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true));
  } else {
    r[0] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, scale, false));
    r[1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, scale, true));
    r[2] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, scale, false));
    r[3] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, scale, true));
  }
  return r;
}
__device__ __forceinline__ float scale_of(unsigned byte) { return __uint_as_float(byte << 23); }

// Result or part of four neighbouring values of a row.
template <bool BF>
__device__ __forceinline__ void store4(char* at, f4v x) {
  *reinterpret_cast<u2v*>(at) = u2v{pack2<BF>(x[0], x[1]), pack2<BF>(x[2], x[3])};
}

__device__ __forceinline__ float over_groups_sum(float x) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_int(x), __float_as_int(x), false, false);
  x = __int_as_float(r[0]) + __int_as_float(r[1]);
  r = __builtin_amdgcn_permlane16_swap(__float_as_int(x), __float_as_int(x), false, false);
  return __int_as_float(r[0]) + __int_as_float(r[1]);
}

// ---------------------------------------------------------------------------
// Attention, blocks of 16 * CB rows.  Work group = 4 waves that share the rows and split the part's keys: units of 32 keys,
// neighbouring ones to a wave, no barrier between them.  A unit comes to registers while the one before is worked on, goes to the
// wave's own tile of LDS (converted there from 8 bits), scores are formed transposed, S^T[keys][rows], so that the 16-bit
// probabilities are the second product's operand as they are (Geom16).  At the end the waves' sums are joined in LDS.
// ---------------------------------------------------------------------------
constexpr int kFewWaves = 4;
constexpr int kUnit = 32;
template <int D, int CB>
struct FewGeom {
  static constexpr int kRows = 16 * CB;
  static constexpr int kTileBytes = kUnit * D * 2;
  static constexpr int kPitch = D * 4 + 16;  // of a row of sums in LDS
  static constexpr int kJoinBytes = kRows * kPitch;
  static constexpr int kWaveBytes = (2 * kTileBytes > kJoinBytes ? 2 * kTileBytes : kJoinBytes + 1023) / 1024 * 1024;
};

template <int D, int CB, bool BF, bool Q8>
__global__ void __launch_bounds__(kFewWaves * 64, 2) paged_few_kernel(PagedArgs a) {
  using T = SwzTile<D>;
  using G = FewGeom<D, CB>;
  constexpr int kRows = G::kRows, kNC = T::kNC, kKS = D / 32, kDB = D / 16;
  constexpr int kLoads = Q8 ? kNC / 2 : kNC;  // of 16 positions: 64 bytes of each
  __shared__ __attribute__((aligned(1024))) char smem[kFewWaves * G::kWaveBytes];
  __shared__ float2 join[kFewWaves][kRows];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int m = lane & 15, g = lane >> 4;
  if (a.zero_rest) {
    const int rest = min(max(a.ends[a.batch - 1], 0), a.tokens);
    const long from = (long)rest * a.head * D * 2, to = (long)a.tokens * a.head * D * 2;
    for (long i = from + ((long)blockIdx.x * blockDim.x + threadIdx.x) * 16; i < to; i += (long)gridDim.x * blockDim.x * 16)
      *reinterpret_cast<u4v*>(a.o + i) = u4v{0, 0, 0, 0};
  }
  const Part w = part_of<kRows>(a, blockIdx.x, lane);
  if (w.b < 0) return;
  const int rows = w.s.n * a.group, row0 = w.block * kRows;
  const int last_token = (min(rows, row0 + kRows) - 1) / a.group;
  const int seen = paged_visible(w.s.keys, w.s.n, last_token, a.causal);
  const int all_see = paged_visible(w.s.keys, w.s.n, row0 / a.group, a.causal);
  int t0, t1;
  paged_part(paged_tiles(seen), w.parts, w.p, t0, t1);
  const int units = min(2 * t1, (seen + kUnit - 1) / kUnit) - 2 * t0;  // of the part
  const int u0 = 2 * t0 + max(units, 0) * wave / kFewWaves, u1 = 2 * t0 + max(units, 0) * (wave + 1) / kFewWaves;

  h8 qf[CB][kKS];
  int sees[CB];  // keys that the lane's row of a column block sees
#pragma unroll
  for (int cb = 0; cb < CB; ++cb) {
    const int row = min(row0 + 16 * cb + m, rows - 1), token = row / a.group, head = row - token * a.group;
    sees[cb] = paged_visible(w.s.keys, w.s.n, token, a.causal);
    const char* at = a.q + w.b * a.q_batch + ((a.ends ? w.s.first : 0) + token) * a.q_seq + (w.head * (int)a.group + head) * a.q_head;
#pragma unroll
    for (int kk = 0; kk < kKS; ++kk) qf[cb][kk] = *reinterpret_cast<const h8*>(at + kk * 64 + g * 16);
  }

  char* const k_tile = smem + wave * G::kWaveBytes;
  char* const v_tile = k_tile + G::kTileBytes;
  const int r16 = lane >> 2, q4 = lane & 3;
  const char* const k_head = a.k + (long)w.head * a.ks.head;
  const char* const v_head = a.v + (long)w.head * a.vs.head;
  const int col = Q8 ? q4 * 16 : (q4 ^ swz(r16 >> 2)) * 16;
  bool bad = w.s.past;
  // page numbers of 64 stretches of 16 positions, from stretch ids0 on
  int ids = 0, ids0 = 0;
  auto fetch_ids = [&](int stretch0) __attribute__((always_inline)) {
    ids0 = stretch0;
    const int at = min((stretch0 + lane) * 16, w.s.keys - 1);
    ids = a.table[w.b * a.table_stride + at / a.page_size];
    const bool none = (unsigned)ids >= (unsigned)a.pages;
    // of stretches that are behind the wave's last one nothing is said
    bad |= __builtin_amdgcn_ballot_w64(none && stretch0 + lane < 2 * u1) != 0;
    if (none) ids = 0;
  };
  u4v kr[2][kLoads], vr[2][kLoads];
  unsigned ksc[2], vsc[2];
  auto load = [&](int u) __attribute__((always_inline)) {
    if (2 * u - ids0 >= 64) fetch_ids(2 * u);
#pragma unroll
    for (int R = 0; R < 2; ++R) {
      const int stretch = min(2 * u + R, (w.s.keys - 1) >> 4);  // positions past the last one: the last one again
      const int pos = stretch * 16, page_at = pos / a.page_size, slot = pos - page_at * a.page_size;
      const long id = __builtin_amdgcn_readlane(ids, stretch - ids0);
      const int r = min(r16, w.s.keys - 1 - pos);
      const char* const kb = k_head + id * a.ks.page + (long)slot * a.ks.slot;
      const char* const vb = v_head + id * a.vs.page + (long)slot * a.vs.slot;
#pragma unroll
      for (int i = 0; i < kLoads; ++i) kr[R][i] = *reinterpret_cast<const u4v*>(kb + (unsigned)(r * a.ks.slot + col + 64 * i));
#pragma unroll
      for (int i = 0; i < kLoads; ++i) vr[R][i] = *reinterpret_cast<const u4v*>(vb + (unsigned)(r * a.vs.slot + col + 64 * i));
      if constexpr (Q8) {
        ksc[R] = a.k_scale[id * a.kss.page + (long)(slot + r) * a.kss.slot + (long)w.head * a.kss.head];
        vsc[R] = a.v_scale[id * a.vss.page + (long)(slot + r) * a.vss.slot + (long)w.head * a.vss.head];
      }
    }
  };
  auto to_lds = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int R = 0; R < 2; ++R) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        if constexpr (Q8) {
          const int at = T::block_off(R, 2 * i + (q4 >> 1)) + r16 * 64;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int chunk = ((2 * (q4 & 1) + e) ^ swz(r16 >> 2)) * 16;
            *reinterpret_cast<u4v*>(k_tile + at + chunk) = from_e4m3<BF>(kr[R][i][2 * e], kr[R][i][2 * e + 1], scale_of(ksc[R]));
            *reinterpret_cast<u4v*>(v_tile + at + chunk) = from_e4m3<BF>(vr[R][i][2 * e], vr[R][i][2 * e + 1], scale_of(vsc[R]));
          }
        } else {
          *reinterpret_cast<u4v*>(k_tile + T::block_off(R, i) + lane * 16) = kr[R][i];
          *reinterpret_cast<u4v*>(v_tile + T::block_off(R, i) + lane * 16) = vr[R][i];
        }
      }
    }
  };

  f4v o[CB][kDB];
  float mc[CB], l[CB];
#pragma unroll
  for (int cb = 0; cb < CB; ++cb) {
    mc[cb] = -INFINITY, l[cb] = 0.f;
#pragma unroll
    for (int db = 0; db < kDB; ++db) o[cb][db] = f4v{0.f, 0.f, 0.f, 0.f};
  }
  const unsigned ka0 = opaque_lds_address(k_tile + rows16_off<D>(lane, 0)), ka1 = opaque_lds_address(k_tile + rows16_off<D>(lane, 1));
  const Cols16<D> va(v_tile, lane);

  if (u0 < u1) {
    fetch_ids(2 * u0);
    load(u0);
  }
  for (int u = u0; u < u1; ++u) {
    to_lds();
    if (u + 1 < u1) load(u + 1);
    f4v s[CB][2];
#pragma unroll
    for (int kk = 0; kk < kKS; ++kk) {
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const h8 kf = rows16_at<D>(ka0, ka1, p, kk);
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) s[cb][p] = mma16<BF>(kf, qf[cb][kk], kk == 0 ? f4v{0.f, 0.f, 0.f, 0.f} : s[cb][p]);
      }
    }
    const int key0 = u * kUnit;
    u4v pf[CB];
    float alpha[CB];
    bool moved = false;
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) {
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = s[cb][e >> 2][e & 3] * a.c;
      if (key0 + kUnit > all_see) {
        const int left = sees[cb] - key0 - 16 * (g >> 1) - 4 * (g & 1);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (8 * (e >> 2) + (e & 3) >= left) x[e] = -INFINITY;
      }
      float mx = x[0];
#pragma unroll
      for (int e = 1; e < 8; ++e) mx = fmaxf(mx, x[e]);
      mx = fmaxf(max_over_groups(mx), mc[cb]);
      const float from = mx == -INFINITY ? 0.f : mx;  // no key yet: every exponential is 0
      alpha[cb] = fast_exp2(mc[cb] - from);
      moved |= mx != mc[cb];
      mc[cb] = mx;
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] = fast_exp2(x[e] - from);
        sum += x[e];
      }
      l[cb] = l[cb] * alpha[cb] + sum;
#pragma unroll
      for (int e = 0; e < 4; ++e) pf[cb][e] = pack2<BF>(x[2 * e], x[2 * e + 1]);
    }
    if (__builtin_amdgcn_ballot_w64(moved)) {
#pragma unroll
      for (int cb = 0; cb < CB; ++cb)
#pragma unroll
        for (int db = 0; db < kDB; ++db) o[cb][db] *= alpha[cb];
    }
#pragma unroll
    for (int db = 0; db < kDB; ++db) {
      const h8 vf = va.at(0, 0, db);
#pragma unroll
      for (int cb = 0; cb < CB; ++cb) o[cb][db] = mma16<BF>(vf, __builtin_bit_cast(h8, pf[cb]), o[cb][db]);
    }
  }

  // the waves' sums, relative to the largest maximum
#pragma unroll
  for (int cb = 0; cb < CB; ++cb) {
    const float sum = over_groups_sum(l[cb]);
    if (g == 0) join[wave][16 * cb + m] = float2{mc[cb], bad ? NAN : sum};
  }
  __syncthreads();
  float* const mine = reinterpret_cast<float*>(smem + wave * G::kWaveBytes);
#pragma unroll
  for (int cb = 0; cb < CB; ++cb) {
    float mx = -INFINITY;
#pragma unroll
    for (int v = 0; v < kFewWaves; ++v) mx = fmaxf(mx, join[v][16 * cb + m].x);
    const float f = mc[cb] == -INFINITY ? 0.f : fast_exp2(mc[cb] - mx);
#pragma unroll
    for (int db = 0; db < kDB; ++db)
      *reinterpret_cast<f4v*>(reinterpret_cast<char*>(mine) + (16 * cb + m) * G::kPitch + db * 64 + g * 16) = o[cb][db] * f;
  }
  __syncthreads();
  constexpr int kPieces = D / 4;  // of a row
  for (int i = threadIdx.x; i < kRows * kPieces; i += kFewWaves * 64) {
    const int row = i / kPieces, piece = i % kPieces;
    if (row0 + row >= rows) break;
    float mx = -INFINITY, sum = 0.f;
#pragma unroll
    for (int v = 0; v < kFewWaves; ++v) mx = fmaxf(mx, join[v][row].x);
    f4v x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int v = 0; v < kFewWaves; ++v) {
      const float2 j = join[v][row];
      sum += j.x == -INFINITY ? j.y : j.y * fast_exp2(j.x - mx);  // without keys 0, or NaN from a bad page
      x += *reinterpret_cast<const f4v*>(smem + v * G::kWaveBytes + row * G::kPitch + piece * 16);
    }
    if (w.parts == 1) {
      const int token = (row0 + row) / a.group, head = w.head * (int)a.group + (row0 + row - token * a.group);
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      store4<BF>(a.o + (((long)(w.s.first + token) * a.head + head) * D + piece * 4) * 2, x * inv);
    } else {
      const long at = (long)w.number * kRows + row;
      *reinterpret_cast<f4v*>(a.part_o + at * D + piece * 4) = x;
      if (piece == 0) a.part_ml[at] = float2{mx, sum};
    }
  }
}

// ---------------------------------------------------------------------------
// Rows whose keys went to several parts.  A work group has one row of the output: D / 4 threads to a part's row.
// ---------------------------------------------------------------------------
template <int D, int ROWS, bool BF>
__global__ void __launch_bounds__(256) paged_join_kernel(PagedArgs a) {
  constexpr int kPieces = D / 4, kSlices = 256 / kPieces;
  __shared__ f4v sums[kSlices][kPieces];
  const int lane = threadIdx.x & 63;
  const int token = (int)blockIdx.x / a.head, head = (int)blockIdx.x - token * a.head;
  const int b = a.ends ? sequence_of(a.ends, a.batch, token, lane) : token / a.new_tokens;
  const Sequence s = sequence(a, b);
  const int i = token - s.first;
  if (i < 0 || i >= s.n) return;
  const int per = tiles_of_part<ROWS>(a, lane);
  const int parts = paged_parts(paged_tiles(s.keys), per);
  if (parts == 1) return;
  int before = 0;
  for (int b0 = lane; b0 < b; b0 += 64) {
    const Sequence t = sequence(a, b0);
    before += paged_blocks(t.n * a.group, ROWS) * paged_parts(paged_tiles(t.keys), per);
  }
  before = (int)sum_over_wave(before);
  const int kvh = head / a.group, row = i * a.group + head - kvh * a.group, block = row / ROWS;
  const long first = (long)before * a.kv_head + ((long)kvh * paged_blocks(s.n * a.group, ROWS) + block) * parts;
  if (first + parts > a.slots) return;
  const long at = first * ROWS + row % ROWS;
  float mx = -INFINITY;
  for (int p = lane; p < parts; p += 64) mx = fmaxf(mx, a.part_ml[at + (long)p * ROWS].x);
#pragma unroll
  for (int d = 1; d < 64; d *= 2) mx = fmaxf(mx, __shfl_xor(mx, d));
  float sum = 0.f;
  for (int p = lane; p < parts; p += 64) {
    const float2 ml = a.part_ml[at + (long)p * ROWS];
    sum += ml.x == -INFINITY ? ml.y : ml.y * fast_exp2(ml.x - mx);
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d);
  const int slice = threadIdx.x / kPieces, piece = threadIdx.x % kPieces;
  f4v x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int p = slice; p < parts; p += kSlices) {
    const float m = a.part_ml[at + (long)p * ROWS].x;
    const f4v y = *reinterpret_cast<const f4v*>(a.part_o + (at + (long)p * ROWS) * D + piece * 4);
    x += y * (m == -INFINITY ? 0.f : fast_exp2(m - mx));
  }
  sums[slice][piece] = x;
  __syncthreads();
  if (slice) return;
#pragma unroll
  for (int v = 1; v < kSlices; ++v) x += sums[v][piece];
  store4<BF>(a.o + (((long)token * a.head + head) * D + piece * 4) * 2, x * (sum == 0.f ? 0.f : 1.f / sum));
}

// ---------------------------------------------------------------------------
// Writing: a wave to a token, its lanes over 16 bytes of all key heads' keys, then values.  Bound by its bytes.
// ---------------------------------------------------------------------------
struct WriteArgs {
  const char *k, *v;
  long k_batch, k_seq, k_head, v_batch, v_seq, v_head;  // bytes
  char *kc, *vc;
  unsigned char *k_scale, *v_scale;
  CacheStrides ks, vs, kss, vss;
  const int *table, *keys, *ends;
  long table_stride;
  int batch, new_tokens, tokens, kv_head, pages, width;
  FmhaDivisor page_size, per_sequence;  // per_sequence: new tokens of each, where ends is null
};

template <bool BF>
__device__ __forceinline__ float to_float(unsigned bits16) {
  if constexpr (BF) return __uint_as_float(bits16 << 16);
  else return (float)__builtin_bit_cast(half_t, (unsigned short)bits16);
}

template <int D, bool BF, bool Q8>
__global__ void __launch_bounds__(256) paged_write_kernel(WriteArgs a) {
  constexpr int kChunks = D / 8;
  const int lane = threadIdx.x & 63, t = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (t >= a.tokens) return;
  int b, i, n;
  if (a.ends) {
    b = __builtin_amdgcn_readfirstlane(sequence_of(a.ends, a.batch, t, lane));
    const int first = min(max(a.ends[b - 1], 0), a.tokens), end = min(max(a.ends[b], first), a.tokens);
    if (t < first || t >= end) return;
    i = t - first, n = end - first;
  } else {
    b = t / a.per_sequence, n = a.per_sequence;
    i = t - b * n;
  }
  const long pos = (long)max(a.keys[b], 0) - n + i;
  if (pos < 0 || pos >= (long)a.width * (int)a.page_size) return;
  const int page_at = (int)pos / a.page_size, slot = (int)pos - page_at * (int)a.page_size;
  const long id = a.table[b * a.table_stride + page_at];
  if (id < 0 || id >= a.pages) return;
  const char* const k = a.k + (a.ends ? t * a.k_seq : b * a.k_batch + i * a.k_seq);
  const char* const v = a.v + (a.ends ? t * a.v_seq : b * a.v_batch + i * a.v_seq);
  char* const kc = a.kc + id * a.ks.page + (long)slot * a.ks.slot;
  char* const vc = a.vc + id * a.vs.page + (long)slot * a.vs.slot;
  for (int e = lane; e < 2 * a.kv_head * kChunks; e += 64) {
    const int r = e / kChunks, chunk = e % kChunks;
    const bool value = r >= a.kv_head;
    const int head = value ? r - a.kv_head : r;
    const u4v x = *reinterpret_cast<const u4v*>((value ? v + head * a.v_head : k + head * a.k_head) + chunk * 16);
    char* const to = value ? vc + (long)head * a.vs.head : kc + (long)head * a.ks.head;
    if constexpr (!Q8) {
      *reinterpret_cast<u4v*>(to + chunk * 16) = x;
    } else {
      const float most = BF ? 0x1.ep127f : 61440.f;
      float y[8], amax = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float z = to_float<BF>(x[j >> 1] >> (16 * (j & 1)) & 0xffff);
        y[j] = z > most ? most : z < -most ? -most : z;  // NaN as it is
        amax = fmaxf(amax, fabsf(z == z ? y[j] : 0.f));
      }
#pragma unroll
      for (int d = 1; d < kChunks; d *= 2) amax = fmaxf(amax, __shfl_xor(amax, d));
      // exponent of 2^e, biased: 448 is 1.75 * 2^8
      const int byte = max((int)((__float_as_uint(amax) + 0x1fffffu) >> 23) - 8, 1);
      const float down = __uint_as_float((unsigned)(254 - byte) << 23);
      u2v out;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * j] * down, y[4 * j + 1] * down, 0, false);
        out[j] = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * j + 2] * down, y[4 * j + 3] * down, w, true);
      }
      *reinterpret_cast<u2v*>(to + chunk * 8) = out;
      if (chunk == 0) {
        unsigned char* const s = value ? a.v_scale + id * a.vss.page + (long)slot * a.vss.slot + (long)head * a.vss.head
                                       : a.k_scale + id * a.kss.page + (long)slot * a.kss.slot + (long)head * a.kss.head;
        *s = (unsigned char)byte;
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Reading: 16 bytes of the result to a lane and step.  Bound by its bytes.
// ---------------------------------------------------------------------------
struct ReadArgs {
  const char *kc, *vc;
  const unsigned char *k_scale, *v_scale;
  char *k, *v;
  CacheStrides ks, vs, kss, vss;
  const int *table, *keys;
  long table_stride;
  int max_seqlen, pages, width;
  FmhaDivisor page_size, kv_head, blocks;  // blocks: work groups of a sequence
};
constexpr int kReadSteps = 8;

template <int D, bool BF, bool Q8>
__global__ void __launch_bounds__(256) paged_read_kernel(ReadArgs a) {
  constexpr int kChunks = D / 8;
  const int w = blockIdx.x, b = w / a.blocks, block = w - b * (int)a.blocks;
  const bool value = blockIdx.y;
  const int keys = max(a.keys[b], 0);
  const char* const cache = value ? a.vc : a.kc;
  const unsigned char* const scales = value ? a.v_scale : a.k_scale;
  const CacheStrides st = value ? a.vs : a.ks, sst = value ? a.vss : a.kss;
  char* const out = (value ? a.v : a.k) + (long)b * a.max_seqlen * (int)a.kv_head * D * 2;
  const int row0 = block * (256 * kReadSteps / kChunks);
#pragma unroll
  for (int u = 0; u < kReadSteps; ++u) {
    const int row = row0 + (u * 256 + threadIdx.x) / kChunks, chunk = threadIdx.x % kChunks;
    const int pos = row / a.kv_head, head = row - pos * (int)a.kv_head;
    if (pos >= a.max_seqlen) continue;
    u4v x = {0, 0, 0, 0};
    if (pos < keys) {
      const int page_at = pos / a.page_size, slot = pos - page_at * (int)a.page_size;
      const long id = page_at < a.width ? a.table[b * a.table_stride + page_at] : -1;
      if (id < 0 || id >= a.pages) {
        x[0] = x[1] = x[2] = x[3] = BF ? 0x7fc07fc0u : 0x7e007e00u;  // NaN
      } else {
        const char* const from = cache + id * st.page + (long)slot * st.slot + (long)head * st.head;
        if constexpr (Q8) {
          const u2v y = *reinterpret_cast<const u2v*>(from + chunk * 8);
          const unsigned s = scales[id * sst.page + (long)slot * sst.slot + (long)head * sst.head];
          x = from_e4m3<BF>(y[0], y[1], scale_of(s));
        } else {
          x = *reinterpret_cast<const u4v*>(from + chunk * 16);
        }
      }
    }
    *reinterpret_cast<u4v*>(out + (long)row * (D * 2) + chunk * 16) = x;
  }
}

// ---------------------------------------------------------------------------
// Host.
// ---------------------------------------------------------------------------
template <typename Args>
hipError_t launch(void (*kernel)(Args), dim3 grid, unsigned block, hipStream_t stream, Args args) {
  void* ptrs[] = {&args};
  return hipLaunchKernel((const void*)kernel, grid, dim3(block), ptrs, 0, stream);
}

bool misaligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; }

// Rows on 16-byte boundaries; offsets inside 16 positions fit 32 bits.
bool bad_strides(const paged_mha_strides& s, int bytes, bool aligned) {
  if (s.page < 0 || s.slot < 0 || s.head < 0 || s.slot >= (1 << 24) || s.head >= (1LL << 30) || s.page >= (1LL << 60)) return true;
  return aligned && (((s.page | s.slot | s.head) * bytes) & 15) != 0;
}
bool bad_strides(const fused_mha_strides* s) {
  if (s->batch < 0 || s->seq < 0 || s->head < 0 || ((s->batch | s->seq | s->head) & 7)) return true;
  return s->batch >= (1LL << 60) || s->seq >= (1LL << 40) || s->head >= (1LL << 40);
}
CacheStrides in_bytes(const paged_mha_strides& s, int bytes) { return {(long)s.page * bytes, (int)(s.slot * bytes), (int)(s.head * bytes)}; }

int check_cache(const paged_mha_cache* c, const paged_mha_batch* b) {
  if (!c || !b || !c->key || !c->value || !b->page_table || !b->cache_seqlens) return FUSED_MHA_ERR_NULL_POINTER;
  if (c->type != PAGED_MHA_FP16 && c->type != PAGED_MHA_BF16) return PAGED_MHA_ERR_BAD_TYPE;
  const bool q8 = c->cache_type == PAGED_MHA_E4M3;
  if (!q8 && c->cache_type != c->type) return PAGED_MHA_ERR_BAD_TYPE;
  if (q8 && (!c->key_scale || !c->value_scale)) return FUSED_MHA_ERR_NULL_POINTER;
  if (!q8 && (c->key_scale || c->value_scale)) return PAGED_MHA_ERR_BAD_TYPE;
  if (c->d != 64 && c->d != 128) return FUSED_MHA_ERR_BAD_HEAD_DIM;
  if (c->pages <= 0 || c->kv_head <= 0 || b->batch <= 0 || b->tokens <= 0 || b->table_width <= 0 || b->table_stride < 0)
    return FUSED_MHA_ERR_BAD_SHAPE;
  if (c->page_size <= 0 || c->page_size % 16) return PAGED_MHA_ERR_BAD_PAGE_SIZE;
  if (c->kv_head > (1 << 16) || b->batch > (1 << 20) || b->table_stride >= (1LL << 40)) return FUSED_MHA_ERR_TOO_LARGE;
  if ((long)b->table_width * c->page_size >= (1L << 30)) return FUSED_MHA_ERR_TOO_LARGE;
  const int bytes = q8 ? 1 : 2;
  if (bad_strides(c->key_strides, bytes, true) || bad_strides(c->value_strides, bytes, true)) return FUSED_MHA_ERR_BAD_STRIDE;
  if (q8 && (bad_strides(c->key_scale_strides, 1, false) || bad_strides(c->value_scale_strides, 1, false))) return FUSED_MHA_ERR_BAD_STRIDE;
  if (misaligned(c->key) || misaligned(c->value)) return FUSED_MHA_ERR_MISALIGNED;
  return FUSED_MHA_OK;
}

long all_tokens(const paged_mha_batch* b) { return b->cu_seqlens ? b->tokens : (long)b->tokens * b->batch; }

// Parts that a launch aims at, and the least tiles of one.
constexpr int kTarget = 512, kLeast = 4;

struct Launch {
  int rows_of_block;
  long items;  // at most
  int target;
  long slots() const { return target ? items + target : 0; }
  long grid() const { return (items + target + 7) / 8 * 8; }
};
Launch plan(const paged_mha_cache* c, const paged_mha_batch* b, int head, int max_new) {
  const long group = head / c->kv_head;
  const long most = b->cu_seqlens ? (max_new > 0 ? std::min<long>(max_new, b->tokens) : b->tokens) : b->tokens;
  Launch p;
  p.rows_of_block = most * group <= 16 ? 16 : 32;
  const long blocks = b->cu_seqlens ? b->tokens * group / p.rows_of_block + b->batch : b->batch * ((b->tokens * group + p.rows_of_block - 1) / p.rows_of_block);
  p.items = blocks * c->kv_head;
  p.target = (long)b->table_width * c->page_size > kLeast * kPagedTile ? kTarget : 0;
  return p;
}
size_t workspace_bytes_of(const Launch& p, int d) { return (size_t)p.slots() * p.rows_of_block * (d * 4 + 8); }

template <int D, int CB, bool BF, bool Q8>
int launch_few(const Launch& p, const PagedArgs& a, hipStream_t stream) {
  if (launch(paged_few_kernel<D, CB, BF, Q8>, dim3(p.grid()), kFewWaves * 64, stream, a) != hipSuccess) return FUSED_MHA_ERR_LAUNCH;
  if (!p.target) return FUSED_MHA_OK;
  const long rows = (long)a.tokens * a.head;
  return launch(paged_join_kernel<D, 16 * CB, BF>, dim3(rows), 256, stream, a) == hipSuccess ? FUSED_MHA_OK : FUSED_MHA_ERR_LAUNCH;
}

// f(D, BF, Q8) with the values of a cache as constants.
template <typename F>
int with_types(const paged_mha_cache* c, F&& f) {
  auto types = [&](auto d) {
    const bool q8 = c->cache_type == PAGED_MHA_E4M3;
    if (c->type == PAGED_MHA_BF16) return q8 ? f(d, IntTag<1>{}, IntTag<1>{}) : f(d, IntTag<1>{}, IntTag<0>{});
    return q8 ? f(d, IntTag<0>{}, IntTag<1>{}) : f(d, IntTag<0>{}, IntTag<0>{});
  };
  return c->d == 64 ? types(IntTag<64>{}) : types(IntTag<128>{});
}

}  // namespace

extern "C" {

int paged_mha_write(const paged_mha_cache* c, const paged_mha_batch* b, const void* k, const fused_mha_strides* k_st, const void* v,
                    const fused_mha_strides* v_st, void* stream) {
  if (const int rc = check_cache(c, b)) return rc;
  if (!k || !v || !k_st || !v_st) return FUSED_MHA_ERR_NULL_POINTER;
  if (bad_strides(k_st) || bad_strides(v_st)) return FUSED_MHA_ERR_BAD_STRIDE;
  if (misaligned(k) || misaligned(v)) return FUSED_MHA_ERR_MISALIGNED;
  const long tokens = all_tokens(b);
  if (tokens >= (1L << 30)) return FUSED_MHA_ERR_TOO_LARGE;
  const int bytes = c->cache_type == PAGED_MHA_E4M3 ? 1 : 2;
  WriteArgs a{};
  a.k = (const char*)k, a.v = (const char*)v;
  a.k_batch = k_st->batch * 2, a.k_seq = k_st->seq * 2, a.k_head = k_st->head * 2;
  a.v_batch = v_st->batch * 2, a.v_seq = v_st->seq * 2, a.v_head = v_st->head * 2;
  a.kc = (char*)c->key, a.vc = (char*)c->value;
  a.k_scale = (unsigned char*)c->key_scale, a.v_scale = (unsigned char*)c->value_scale;
  a.ks = in_bytes(c->key_strides, bytes), a.vs = in_bytes(c->value_strides, bytes);
  a.kss = in_bytes(c->key_scale_strides, 1), a.vss = in_bytes(c->value_scale_strides, 1);
  a.table = b->page_table, a.keys = b->cache_seqlens, a.ends = b->cu_seqlens ? b->cu_seqlens + 1 : nullptr;
  a.table_stride = b->table_stride;
  a.batch = b->batch, a.tokens = (int)tokens;
  a.kv_head = c->kv_head, a.pages = c->pages, a.width = b->table_width;
  a.page_size = FmhaDivisor(c->page_size), a.per_sequence = FmhaDivisor(b->tokens);
  return with_types(c, [&](auto d, auto bf, auto q8) {
    const auto kernel = paged_write_kernel<decltype(d)::value, decltype(bf)::value != 0, decltype(q8)::value != 0>;
    return launch(kernel, dim3((tokens + 3) / 4), 256, (hipStream_t)stream, a) == hipSuccess ? FUSED_MHA_OK : FUSED_MHA_ERR_LAUNCH;
  });
}

int paged_mha_read(const paged_mha_cache* c, const paged_mha_batch* b, int max_seqlen, void* k, void* v, void* stream) {
  if (const int rc = check_cache(c, b)) return rc;
  if (!k || !v) return FUSED_MHA_ERR_NULL_POINTER;
  if (misaligned(k) || misaligned(v)) return FUSED_MHA_ERR_MISALIGNED;
  if (max_seqlen <= 0) return FUSED_MHA_ERR_BAD_SHAPE;
  const int rows_of_block = 256 * kReadSteps / (c->d / 8);
  const long rows = (long)max_seqlen * c->kv_head, blocks = (rows + rows_of_block - 1) / rows_of_block;
  if (rows >= (1L << 30) || blocks * b->batch >= (1L << 30)) return FUSED_MHA_ERR_TOO_LARGE;
  const int bytes = c->cache_type == PAGED_MHA_E4M3 ? 1 : 2;
  ReadArgs a{};
  a.kc = (const char*)c->key, a.vc = (const char*)c->value;
  a.k_scale = (const unsigned char*)c->key_scale, a.v_scale = (const unsigned char*)c->value_scale;
  a.k = (char*)k, a.v = (char*)v;
  a.ks = in_bytes(c->key_strides, bytes), a.vs = in_bytes(c->value_strides, bytes);
  a.kss = in_bytes(c->key_scale_strides, 1), a.vss = in_bytes(c->value_scale_strides, 1);
  a.table = b->page_table, a.keys = b->cache_seqlens, a.table_stride = b->table_stride;
  a.max_seqlen = max_seqlen, a.pages = c->pages, a.width = b->table_width;
  a.page_size = FmhaDivisor(c->page_size), a.kv_head = FmhaDivisor(c->kv_head), a.blocks = FmhaDivisor((int)blocks);
  return with_types(c, [&](auto d, auto bf, auto q8) {
    const auto kernel = paged_read_kernel<decltype(d)::value, decltype(bf)::value != 0, decltype(q8)::value != 0>;
    return launch(kernel, dim3(blocks * b->batch, 2), 256, (hipStream_t)stream, a) == hipSuccess ? FUSED_MHA_OK : FUSED_MHA_ERR_LAUNCH;
  });
}

static int check_forward(const paged_mha_cache* c, const paged_mha_batch* b, int head, int max_new) {
  if (const int rc = check_cache(c, b)) return rc;
  if (head <= 0 || max_new < 0) return FUSED_MHA_ERR_BAD_SHAPE;
  if (head % c->kv_head) return PAGED_MHA_ERR_BAD_GROUP;
  if (head > (1 << 16) || all_tokens(b) * head >= (1L << 30)) return FUSED_MHA_ERR_TOO_LARGE;
  return plan(c, b, head, max_new).grid() >= (1L << 30) ? FUSED_MHA_ERR_TOO_LARGE : FUSED_MHA_OK;
}

size_t paged_mha_forward_workspace_bytes(const paged_mha_cache* c, const paged_mha_batch* b, int head, int max_new) {
  return check_forward(c, b, head, max_new) ? 0 : workspace_bytes_of(plan(c, b, head, max_new), c->d);
}

int paged_mha_forward(const paged_mha_cache* c, const paged_mha_batch* b, const void* q, const fused_mha_strides* q_st, void* o,
                      int head, int max_new, float scale, int causal, int zero_rest, void* workspace, size_t workspace_bytes,
                      void* stream) {
  if (const int rc = check_forward(c, b, head, max_new)) return rc;
  if (!q || !q_st || !o) return FUSED_MHA_ERR_NULL_POINTER;
  if (!isfinite(scale)) return FUSED_MHA_ERR_BAD_SCALE;
  if (bad_strides(q_st)) return FUSED_MHA_ERR_BAD_STRIDE;
  const Launch p = plan(c, b, head, max_new);
  const size_t wanted = workspace_bytes_of(p, c->d);
  if (wanted && !workspace) return FUSED_MHA_ERR_NULL_POINTER;
  if (workspace_bytes < wanted) return PAGED_MHA_ERR_WORKSPACE;
  if (misaligned(q) || misaligned(o) || misaligned(workspace)) return FUSED_MHA_ERR_MISALIGNED;
  const int bytes = c->cache_type == PAGED_MHA_E4M3 ? 1 : 2;
  PagedArgs a{};
  a.q = (const char*)q, a.k = (const char*)c->key, a.v = (const char*)c->value, a.o = (char*)o;
  a.k_scale = (const unsigned char*)c->key_scale, a.v_scale = (const unsigned char*)c->value_scale;
  a.table = b->page_table, a.keys = b->cache_seqlens, a.ends = b->cu_seqlens ? b->cu_seqlens + 1 : nullptr;
  a.part_o = (float*)workspace;
  a.part_ml = (float2*)((char*)workspace + (size_t)p.slots() * p.rows_of_block * c->d * 4);
  a.ks = in_bytes(c->key_strides, bytes), a.vs = in_bytes(c->value_strides, bytes);
  a.kss = in_bytes(c->key_scale_strides, 1), a.vss = in_bytes(c->value_scale_strides, 1);
  a.q_batch = a.ends ? 0 : q_st->batch * 2, a.q_seq = q_st->seq * 2, a.q_head = q_st->head * 2;
  a.table_stride = b->table_stride;
  a.batch = b->batch, a.new_tokens = b->tokens, a.tokens = (int)all_tokens(b);
  a.head = head, a.kv_head = c->kv_head, a.pages = c->pages, a.width = b->table_width;
  a.group = FmhaDivisor(head / c->kv_head), a.page_size = FmhaDivisor(c->page_size);
  a.c = scale * kLog2e;
  a.causal = causal != 0, a.zero_rest = zero_rest != 0 && a.ends;
  a.target = p.target, a.least = kLeast, a.slots = (int)p.slots();
  return with_types(c, [&](auto d, auto bf, auto q8) {
    constexpr int D = decltype(d)::value;
    constexpr bool BF = decltype(bf)::value != 0, Q8 = decltype(q8)::value != 0;
    return p.rows_of_block == 16 ? launch_few<D, 1, BF, Q8>(p, a, (hipStream_t)stream) : launch_few<D, 2, BF, Q8>(p, a, (hipStream_t)stream);
  });
}

const char* paged_mha_error_string(int code) {
  switch (code) {
    case FUSED_MHA_OK: return "success";
    case FUSED_MHA_ERR_NULL_POINTER: return "a required pointer is null";
    case FUSED_MHA_ERR_BAD_SHAPE: return "a size is not positive";
    case FUSED_MHA_ERR_BAD_HEAD_DIM: return "head size must be 64 or 128";
    case FUSED_MHA_ERR_MISALIGNED: return "a pointer is not 16-byte aligned";
    case FUSED_MHA_ERR_LAUNCH: return "the HIP runtime refused the launch";
    case FUSED_MHA_ERR_BAD_SCALE: return "softmax scale must be finite";
    case FUSED_MHA_ERR_TOO_LARGE: return "the problem is too large";
    case FUSED_MHA_ERR_BAD_STRIDE: return "strides must be non-negative, with rows on 16-byte boundaries";
    case PAGED_MHA_ERR_BAD_TYPE: return "types must be fp16 or bf16, the cache of the same type or e4m3 with scales";
    case PAGED_MHA_ERR_BAD_PAGE_SIZE: return "page size must be a multiple of 16";
    case PAGED_MHA_ERR_BAD_GROUP: return "query heads must be a multiple of key heads";
    case PAGED_MHA_ERR_WORKSPACE: return "the workspace is too small";
    default: return "unknown error";
  }
}

}  // extern "C"
