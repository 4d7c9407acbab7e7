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
  float* part_o;                   // of each place (paged_place): a block's rows x D sums, relative to the maximum
  float2* part_ml;                 // maximum (of exponents of 2) and sum of each row
  int2* places;                    // of each row of o: its row in place 2 r if its item begins in stretch r, and how many parts it has
  CacheStrides ks, vs, kss, vss;
  long q_batch, q_seq, q_head, table_stride;  // of q in bytes
  int batch, new_tokens, tokens;              // new_tokens: of each sequence, where ends is null; tokens: in all
  int head, pages, width;
  FmhaDivisor kv_head, group, page_size;  // group: query heads of a key head
  float c;                       // scale * log2(e)
  int causal, zero_rest;
  int shared;   // items are shared out (paged_plan.h), otherwise each has a work group
  int step[2];  // of PagedLine under causal masking, for blocks of few rows and of many
  int k_shift, v_shift;  // offsets of 16 positions in the cache are multiples of 2^shift bytes, fewer than 2^32
};

// Says that a pointer is to global memory, which the compiler knows of a kernel's parameters alone: without it loads are flat ones,
// for which every wait for LDS waits too.
template <typename T>
__device__ __forceinline__ void in_global(T*& p) { p = (T*)(__attribute__((address_space(1))) T*)(uintptr_t)p; }

// The kernel's arguments as they lie in memory, asked for where they are needed again: kept in registers across a main loop they
// are spilled.
__device__ __forceinline__ PagedArgs args_again() {
  typedef __attribute__((address_space(4))) const unsigned Word;
  Word* from = (Word*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(from));
  struct Words {
    unsigned w[sizeof(PagedArgs) / 4];
  } words;
#pragma unroll
  for (unsigned i = 0; i < sizeof(PagedArgs) / 4; ++i) words.w[i] = from[i];
  PagedArgs a = __builtin_bit_cast(PagedArgs, words);
  in_global(a.q), in_global(a.k), in_global(a.v), in_global(a.k_scale), in_global(a.v_scale), in_global(a.o), in_global(a.table);
  in_global(a.keys), in_global(a.ends), in_global(a.part_o), in_global(a.part_ml), in_global(a.places);
  return a;
}

// A word of each 64 bytes of them, asked for at once: later loads find them in the scalar cache.
__device__ __forceinline__ void touch_args() {
  typedef __attribute__((address_space(4))) const unsigned Word;
  Word* from = (Word*)__builtin_amdgcn_kernarg_segment_ptr();
  static_assert(sizeof(PagedArgs) > 256 && sizeof(PagedArgs) <= 320, "five of them");
  const unsigned w0 = from[0], w1 = from[16], w2 = from[32], w3 = from[48], w4 = from[64];
  asm volatile("" ::"s"(w0), "s"(w1), "s"(w2), "s"(w3), "s"(w4));
}

struct Sequence {
  int first, n;  // its tokens
  int keys;
  int past;      // it has more keys than the page table has places
};
__device__ __forceinline__ Sequence sequence(const PagedArgs& a, int b) {
  Sequence s;
  const int keys = max(a.keys[b], 0);
  if (a.ends) {
    const int lo = a.ends[b - 1], hi = a.ends[b];
    s.first = min(max(lo, 0), a.tokens);
    s.n = min(max(hi, s.first), a.tokens) - s.first;
  } else {
    s.first = b * a.new_tokens;
    s.n = a.new_tokens;
  }
  const int places = a.width * (int)a.page_size;  // below 2^30
  s.past = keys > places;
  s.keys = min(keys, places);
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

// The same address in all lanes, as the copies want it.
__device__ __forceinline__ const half_t* wave_uniform(const char* p) {
  const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)p);
  const unsigned hi = __builtin_amdgcn_readfirstlane((unsigned)((uintptr_t)p >> 32));
  return (const half_t*)(((uintptr_t)hi << 32) | lo);
}

// The value of one lane.
__device__ __forceinline__ long of_lane(long x, int lane) {
  const unsigned lo = __builtin_amdgcn_readlane((unsigned)x, lane), hi = __builtin_amdgcn_readlane((unsigned)((unsigned long)x >> 32), lane);
  return (long)(((unsigned long)hi << 32) | lo);
}
// Says that all lanes have the same value, which then takes a scalar register.
__device__ __forceinline__ int same(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ float same(float x) { return __int_as_float(same(__float_as_int(x))); }
__device__ __forceinline__ long same(long x) { return of_lane(x, 0); }

// The sum over lanes 0 .. the lane's own, by moves inside rows of 16 lanes and of the last lane of a row, or of two, to the next.
template <int kMove, int kRows>
__device__ __forceinline__ long moved(long x) {
  const unsigned lo = __builtin_amdgcn_update_dpp(0, (int)x, kMove, kRows, 15, false);
  const unsigned hi = __builtin_amdgcn_update_dpp(0, (int)((unsigned long)x >> 32), kMove, kRows, 15, false);
  return (long)(((unsigned long)hi << 32) | lo);
}
__device__ __forceinline__ int scan_over_wave(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 15, 15, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 15, 15, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 15, 15, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 15, 15, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 10, 15, false);  // lane 15 of rows 0 and 2 to rows 1 and 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 12, 15, false);  // lane 31 to rows 2 and 3
  return x;
}
__device__ __forceinline__ long scan_over_wave(long x) {
  x += moved<0x111, 15>(x);
  x += moved<0x112, 15>(x);
  x += moved<0x114, 15>(x);
  x += moved<0x118, 15>(x);
  x += moved<0x142, 10>(x);
  x += moved<0x143, 12>(x);
  return x;
}

// Which blocks a launch has: FEW rows for sequences that have at most kFewRows of them, kManyRows for the others; or all of one
// kind, with FEW = 0 or MANY = false.  A block of many rows multiplies 128 whatever it has, one of few reads its keys for 16 or 32.
// us of 16 sequences of about 4096 keys, 8 key heads of 128, bf16, in blocks of few rows and of many: 32 rows a key head 57.3, 63.0; 48
// 79.5, 64.3; 64 81.2, 65.7.  In blocks of 16 and of 32: 4 rows 49.0, 50.5; of 8 sequences 24.2, 25.9; 200 over 200 keys 26.9, 30.5.
constexpr int kFewRows = 32, kManyRows = 128;
template <int FEW, bool MANY, bool Q8>
struct Blocks {
  static constexpr int kMost = MANY ? kManyRows : FEW;  // rows of a slot
  static __device__ __forceinline__ bool many(int rows) { return MANY && (FEW == 0 || rows > kFewRows); }
  static __device__ __forceinline__ int rows_of_block(int rows) { return many(rows) ? kManyRows : FEW; }
  static __device__ __forceinline__ int count(int rows) { return paged_blocks(rows, rows_of_block(rows)); }
  // The rest is what is known about time, for sharing it out, timed over 20 batches; figures are us.
  // What an item costs beside its keys, in keys: about three tiles where a block has many rows, one where it has few.
  static __device__ __forceinline__ int overhead(int rows) { return many(rows) ? 192 : 64; }
  // Weight of a key: 4 for a block of many rows while another shares its CU, and for one of few, which waits for memory; out of 8 bits
  // that takes half as long.  With 2 and 4 for few rows, a chunk of 512 new tokens beside 39 sequences with one, 4000 keys: 16-bit
  // 105.0, 83.1; 8-bit 69.5, 91.0; two of 500 beside 28 of 8000: 208.2, 170.5; 8-bit 153.8, 159.9.
  static __device__ __forceinline__ int of_key(int rows) { return MANY && FEW && Q8 && !many(rows) ? 2 : 4; }
  // A block of many rows alone on its CU takes 0.58 of the time (one of few as long as with another).  With 0.5, 0.58 and 0.7: 512 new
  // tokens of 8192 88.0, 85.5, 85.6; 900 of 4000 72.9, 71.5, 79.3; three of 300 of 4000 74.0, 73.3, 82.2; 8-bit 91.3, 90.8, 91.4.
  static constexpr float kAlone = MANY ? 0.58f : 1.f;
  // What parts cost (256: a tile): an item more in a stretch, and of many rows to write their sums and to read them again, of up
  // to two in each stretch or of one.  Stretches: few rows with 2, 3 and 6 tiles 16 sequences of 4096 50.5, 49.0, 49.0; of 32 rows 62.2,
  // 57.3, 57.7; many with 8, 17 and 30 900 of 4000 85.8, 71.5, 71.3.  Parts with 2, 6 and 12: 900 of 4000 78.2, 71.5, 71.4; 512 of 8192
  // 85.4, 85.5, 87.5; four of 200 of 2000 52.2, 43.2, 43.0.
  static constexpr float kStretchesCost = (MANY ? 3 + 14 : 3) * 256, kPartsCost = MANY ? 6 * 256 : 0;
};
// What a work group does of an item.
struct Part {
  int b, head, block;
  int t0, t1;        // tiles
  bool whole;        // the item is not in other stretches too
  bool opens;        // it begins here
  int place, parts;  // of the part's sums; of the item
  int stretch;
  Sequence s;
};

// What stands for a token's row that has no score above -inf: 0 if it sees no key, `other` if all that it sees have a score of -inf,
// over which a softmax is NaN.
__device__ __forceinline__ float of_no_score(const Part& w, int token, bool causal, float other) {
  return paged_visible(w.s.keys, w.s.n, token, causal) > 0 ? other : 0.f;
}

__device__ __forceinline__ float max_over_wave(float x) {
  auto turned = [](float y, auto by) __attribute__((always_inline)) {  // inside rows of 16 lanes
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(y), 0x120 + decltype(by)::value, 15, 15, true));
  };
  x = fmaxf(x, turned(x, IntTag<8>{}));
  x = fmaxf(x, turned(x, IntTag<4>{}));
  x = fmaxf(x, turned(x, IntTag<2>{}));
  x = fmaxf(x, turned(x, IntTag<1>{}));
  return max_over_groups(x);
}
// A whole number below 2^62 as a float, and a quotient: nearly, and the same in all work groups.
__device__ __forceinline__ float nearly(long x) { return fmaf((float)(unsigned)((unsigned long)x >> 32), 4294967296.f, (float)(unsigned)x); }
__device__ __forceinline__ float nearly(float x, float y) { return x * __builtin_amdgcn_rcpf(y); }

// A work group's items, one after the other (ways to share them: paged_plan.h); all lanes together, each with one of 64 sequences
// in its registers.  Every work group finds its own from the lengths of all sequences, in about 2700 cycles and 1900 for an item; that
// is time during which no memory is read, so whole numbers of 32 bits serve wherever they can.
// us with stretches, parts, whole items and the way taken: 8 sequences of 4096 keys, 4 rows a key head 24.9, 23.9, 33.9, 24.2; 40 of 3000
// 78.8, 86.1, 96.1, 79.5; 512 new tokens of 8192 94.2, 85.5, 114.8, 85.5; 2048 of as many 76.5, 57.3, 50.1, 52.0; 731 beside single tokens,
// 8-bit, 113.3, 141.0, 99.9, 100.9.
template <typename B>
struct Walk {
  enum Way { kStretches, kParts, kWhole };
  Way way;
  int b0;  // the first of the 64 sequences
  Sequence mine;
  // kParts and kWhole, where an item has `parts` places in a line of them
  int at, items, round;
  int upto, parts;  // the line up to the end of the lane's sequence; of an item of the lane's sequence
  // kStretches
  long x, end, length;  // position; end of the stretch and its length
  long line_upto;
  int stretch;
  __device__ __forceinline__ static PagedLine weights(const PagedArgs& a, int n, int keys) {
    const int rows = n * a.group;
    return paged_line(keys, n, a.group, a.causal ? a.step[B::many(rows)] : 0, B::rows_of_block(rows), B::overhead(rows), B::of_key(rows));
  }
  __device__ __forceinline__ static float heaviest(const PagedArgs& a, int n, int keys) {
    const int rows = n * a.group;
    return n == 0 ? 0.f : (float)B::of_key(rows) * (float)(keys + B::overhead(rows));  // past 32 bits
  }
  __device__ __forceinline__ void load(const PagedArgs& a, int from, int lane) {
    b0 = from;
    mine = sequence(a, min(b0 + lane, a.batch - 1));
  }
  __device__ __forceinline__ void scan(const PagedArgs& a, int before, int lane) {  // not of kStretches
    upto = before + scan_over_wave(b0 + lane < a.batch ? B::count(mine.n * a.group) * (int)a.kv_head * parts : 0);
  }
  __device__ __forceinline__ void scan(const PagedArgs& a, long before, int lane) {
    line_upto = before + scan_over_wave(b0 + lane < a.batch ? weights(a, mine.n, mine.keys).all() * a.kv_head : 0);
  }
  // Finds work group w's first item; false if it has none.
  __device__ __forceinline__ bool begin(const PagedArgs& a, int w, int lane) {
    way = kWhole;
    parts = 1, round = 0, stretch = 0;
    x = end = length = line_upto = 0;
    if (!a.shared && !a.ends) {  // as many items for each sequence: no need to look at others
      const int each = B::count(a.new_tokens * a.group) * a.kv_head;
      items = each * a.batch;
      if (w >= items) return false;
      const int b = same(w / each);
      load(a, b, lane);
      upto = (b + 1) * each;
      at = w;
      return true;
    }
    load(a, 0, lane);
    const bool one = a.batch <= 64;
    scan(a, 0, lane);
    items = __builtin_amdgcn_readlane(upto, 63);
    if (!one) {
      int more = 0;
      for (int b = 64 + lane; b < a.batch; b += 64) more += B::count(sequence(a, b).n * a.group) * (int)a.kv_head;
      items += __builtin_amdgcn_readlane(scan_over_wave(more), 63);
    }
    if (!a.shared) {
      at = w;
      return at < items;
    }
    long all = 0;
    float heavy = 0.f, light = -INFINITY;  // light: less than 0, the least weight
    for (int b = lane; b < a.batch; b += 64) {
      const Sequence s = one ? mine : sequence(a, b);
      const PagedLine t = weights(a, s.n, s.keys);
      all += t.all() * a.kv_head;
      heavy = fmaxf(heavy, heaviest(a, s.n, s.keys));
      if (s.n) light = fmaxf(light, -nearly(t.of(0)));
    }
    all = of_lane(scan_over_wave(all), 63);
    heavy = same(max_over_wave(heavy));
    light = -same(max_over_wave(light));
    const long even = paged_stretch(all);
    const float even_long = nearly(even);
    const int rounds = (items + kPagedGroups - 1) >> kPagedGroupsLog;
    float best = rounds > 1 ? (float)rounds * nearly(nearly(all), (float)items)
                            : fmaxf(B::kAlone * heavy, items <= kCus ? 0.f : 0.5f * (heavy + light));
    if (even_long + B::kStretchesCost < best) {
      best = even_long + B::kStretchesCost;
      way = kStretches;
    }
    int places = 0;
    if (one && items <= kPagedGroups) {
      // 64 lengths, from the even one up to five times that, by as many lanes: the best for which there are stretches enough
      const float mine_long = even_long * (1.f + lane * (1.f / 16.f)), mine_in = __builtin_amdgcn_rcpf(mine_long);
      const float weight = heaviest(a, mine.n, mine.keys);
      const int of_mine = lane < a.batch ? B::count(mine.n * a.group) * (int)a.kv_head : 0;
      int count = 0;
#pragma unroll 8
      for (int b = 0; b < (a.batch + 7) / 8 * 8; ++b)
        count += __builtin_amdgcn_readlane(of_mine, b) * paged_parts(__uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(weight), b)), mine_in);
      const float cost = count <= kCus ? B::kAlone * mine_long + 0.5f * B::kPartsCost : count <= kPagedGroups ? mine_long + B::kPartsCost : INFINITY;
      const float least = -same(max_over_wave(-cost));
      if (least < best) {
        const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(cost == least));
        way = kParts;
        places = __builtin_amdgcn_readlane(count, l);
        parts = paged_parts(weight, __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(mine_in), l)));
        scan(a, 0, lane);
      }
    }
    way = (Way)same((int)way);
    if (way == kStretches) {
      scan(a, 0l, lane);
      length = same(even);
      stretch = same(paged_spread(w, paged_stretches(all, length)));
      x = same(stretch * length);
      end = same(min(x + length, all));
      return x < end;
    }
    at = same(way == kParts ? paged_spread(w, places) : paged_whole(0, w, items));
    return at < (way == kParts ? places : items);
  }
  __device__ __forceinline__ bool more() const { return way == kStretches ? x < end : way == kWhole && at < items; }
  __device__ __forceinline__ bool next(const PagedArgs& a, int lane, Part& r) {
    unsigned long long past;
    while (!(past = __builtin_amdgcn_ballot_w64(way == kStretches ? line_upto > x : upto > at))) {
      if (b0 + 64 >= a.batch) return false;
      const long line_before = of_lane(line_upto, 63);
      const int before = __builtin_amdgcn_readlane(upto, 63);
      load(a, b0 + 64, lane);
      if (way == kStretches) scan(a, line_before, lane);
      else scan(a, before, lane);
    }
    const int l = __builtin_ctzll(past);
    r.b = b0 + l;
    r.s.first = __builtin_amdgcn_readlane(mine.first, l);
    r.s.n = __builtin_amdgcn_readlane(mine.n, l);
    r.s.keys = __builtin_amdgcn_readlane(mine.keys, l);
    r.s.past = __builtin_amdgcn_readlane(mine.past, l);
    const int rows = r.s.n * a.group, blocks = B::count(rows), rows_of_block = B::rows_of_block(rows);
    auto scalar = [](int x) __attribute__((always_inline)) { return same(x); };
    if (way != kStretches) {
      const int each = __builtin_amdgcn_readlane(parts, l);
      const int local = at - (__builtin_amdgcn_readlane(upto, l) - blocks * each * (int)a.kv_head);
      int part = 0;
      if (way == kWhole) paged_whole_item(local, blocks, a.kv_head, r.block, r.head);
      else paged_part_item(local, blocks, each, r.block, r.head, part, scalar);
      r.block = same(r.block), r.head = same(r.head);
      const int tiles = paged_tiles_of(r.s.keys, r.s.n, a.group, rows_of_block, r.block, a.causal);
      const float per = (float)tiles * __builtin_amdgcn_rcpf((float)each);
      r.t0 = same(paged_part_tile(tiles, part, each, per));
      r.t1 = same(paged_part_tile(tiles, part + 1, each, per));
      r.opens = part == 0;
      r.whole = each == 1;
      r.parts = each;
      r.place = paged_place(at - part, part);
      r.stretch = at;
      at = way == kWhole && a.shared ? same(paged_whole(++round, blockIdx.x, items)) : items;
      return true;
    }
    const PagedLine line = weights(a, r.s.n, r.s.keys);
    PagedShare share;
    paged_item_at(line, of_lane(line_upto, l) - line.all() * a.kv_head, x, share, scalar);
    const int tiles = paged_tiles_of(r.s.keys, r.s.n, a.group, rows_of_block, share.block, a.causal);
    paged_share_of_stretch(tiles, x, end, length, stretch, share, scalar);
    r.head = share.head, r.block = share.block, r.t0 = share.t0, r.t1 = share.t1;
    r.opens = share.opens, r.whole = share.whole, r.parts = share.parts, r.place = share.place;
    r.stretch = stretch;
    x = same(share.item + share.weight);
    return true;
  }
};

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

template <bool BF>
__device__ __forceinline__ float to_float(unsigned bits16) {
  if constexpr (BF) return __uint_as_float(bits16 << 16);
  else return (float)__builtin_bit_cast(half_t, (unsigned short)bits16);
}

// A key that a row does not see has a probability of 0, which is not enough where its value is infinite or NaN: 0 times that is NaN.
// So in a tile with such keys values are looked at; where some are not finite, only the numbers are multiplied, and the others are
// added in the end to the rows that see them, one key after the other.  What is done with such values is said to be unlikely, so that it
// lies behind the rest of the code.  us without looking and with it: 8 sequences of 3000 keys, 5 tokens of 32 heads of 128, 25.9, 26.4 (26.9
// with that code in between); 2 of 2048 keys, all new, 16 heads of 128, 54.5, 55.7, out of 8 bits 64.6, 66.3; 64 of 64 keys, 40 tokens of
// 8 heads of 64, a tile each, 8.8, 9.2; 512 tokens of 8192 88.2, 88.0, and with an infinity in the last key's value 143; the 5 tokens then 53.
typedef unsigned short us2 __attribute__((ext_vector_type(2)));
template <bool BF>
struct Finite {
  static constexpr unsigned kInf = BF ? 0x7f80 : 0x7c00;
  us2 most = {0, 0};  // of the magnitudes' bits
  __device__ __forceinline__ void look(u4v w) {
#pragma unroll
    for (int i = 0; i < 4; ++i) most = __builtin_elementwise_max(most, __builtin_bit_cast(us2, w[i] & 0x7fff7fffu));
  }
  __device__ __forceinline__ bool all() const {  // of the wave
    return __builtin_amdgcn_ballot_w64(most[0] >= kInf || most[1] >= kInf) == 0;
  }
  __device__ __forceinline__ static u4v numbers(u4v w) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if ((w[i] & 0x7fffu) >= kInf) w[i] &= 0xffff0000u;
      if ((w[i] >> 16 & 0x7fffu) >= kInf) w[i] &= 0xffffu;
    }
    return w;
  }
  // a sum of numbers with a value, given by its 16 bits, if that is not one
  __device__ __forceinline__ static float with_other(float sum, unsigned bits) { return (bits & 0x7fffu) >= kInf ? sum + to_float<BF>(bits) : sum; }
};
// The value of a key: its row in the cache, and out of 8 bits its scale.
struct ValueRow {
  const char* at;  // null: on a page that is none of the cache's
  float scale;
};
template <bool Q8>
__device__ __forceinline__ ValueRow value_row(const PagedArgs& a, const Part& w, int key) {
  const int page_at = key / a.page_size, slot = key - page_at * (int)a.page_size, id = a.table[w.b * a.table_stride + page_at];
  if ((unsigned)id >= (unsigned)a.pages) return ValueRow{nullptr, 0.f};
  return ValueRow{a.v + id * a.vs.page + (long)slot * a.vs.slot + (long)w.head * a.vs.head,
                  Q8 ? scale_of(a.v_scale[id * a.vss.page + (long)slot * a.vss.slot + (long)w.head * a.vss.head]) : 1.f};
}
// Four neighbouring ones of its 16-bit values.
template <bool BF, bool Q8>
__device__ __forceinline__ u2v values4(const char* row, int feature, float scale) {
  if constexpr (!Q8) return *reinterpret_cast<const u2v*>(row + feature * 2);
  const u4v x = from_e4m3<BF>(*reinterpret_cast<const unsigned*>(row + feature), 0, scale);
  return u2v{x[0], x[1]};
}

__device__ __forceinline__ float over_groups_sum(float x) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_int(x), __float_as_int(x), false, false);
  x = __int_as_float(r[0]) + __int_as_float(r[1]);
  r = __builtin_amdgcn_permlane16_swap(__float_as_int(x), __float_as_int(x), false, false);
  return __int_as_float(r[0]) + __int_as_float(r[1]);
}

// ---------------------------------------------------------------------------
// Attention, blocks of 16 * CB rows.  Work group = 4 waves that share the rows and split the part's keys: units of 32 keys,
// neighbouring ones to a wave, no barrier between them, a tile of LDS for each wave.  Scores are formed transposed,
// S^T[keys][rows], so that the 16-bit probabilities are the second product's operand as they are (Geom16).  At the end the waves'
// sums are joined in LDS.
//
// Bound by reading the cache, and for short ones by what waits for what: lengths, pages, keys, the sums of the parts.  4 rows a key
// head, 8 key heads of 128: 131072 keys of one sequence 104 us, 5.2 TB/s of 6.0 that reads alone reach; 8 of about 4096 24.8 us, 3.7 TB/s,
// of which 4.5 for the join; 32 of 8192 in 8 bits 79 us, 4.0 TB/s, where the copies by themselves take 76 (128 bytes of each KiB at a time).
//
// 16-bit cache: a unit comes to registers while the one before is worked on, then goes to the tile.
// 8-bit cache: units are copied to LDS as they are, two at a time, and converted where they become operands.  Keys' scales go into
// the conversion.  Values' scales, which differ along the second product's sum, go into the probabilities: exp2(t + e - m') with
// the value's exponent e and a maximum m' of its own of t + e, so that what counts most is 1 whatever the scales are; in fp16 2^14,
// which leaves values of up to 2^-28 of the largest scale their probabilities' 11 bits, and drops none before 2^-39.
// ---------------------------------------------------------------------------
constexpr int kPagedThreads = 256;
constexpr int kFewWaves = kPagedThreads / 64;
constexpr int kUnit = 32;
template <int D, int CB, bool Q8>
struct FewGeom {
  static constexpr int kRows = 16 * CB;
  static constexpr int kTileBytes = kUnit * D * (Q8 ? 1 : 2);                 // of keys or values
  static constexpr int kSlotBytes = 2 * kTileBytes + (Q8 ? 2 * kUnit * 4 : 0);  // and their scales
  static constexpr int kSlots = Q8 ? 2 : 1;
  static constexpr int kPitch = D * 4 + 16;  // of a row of sums in LDS
  static constexpr int kJoinBytes = kRows * kPitch;
  static constexpr int kWaveBytes = ((kSlots * kSlotBytes > kJoinBytes ? kSlots * kSlotBytes : kJoinBytes) + 1023) / 1024 * 1024;
};

// A byte for each lane to the lane's dword from `lds` on, past the compiler's wait counts like copy16.
__device__ __forceinline__ void copy_byte(const unsigned char* from, unsigned lds) {
  unsigned saved_m0;
  asm volatile(
      "s_mov_b32 %0, m0\n\t"
      "s_mov_b32 m0, %2\n\t"
      "s_nop 0\n\t"
      "global_load_lds_ubyte %1, off\n\t"
      "s_mov_b32 m0, %0"
      : "=&s"(saved_m0)
      : "v"(from), "s"(lds)
      : "memory");
}

template <int D, int CB, bool BF, bool Q8>
__device__ __forceinline__ void few_rows(const PagedArgs& a, const Part& w, char* smem, int slot_rows) {
  using T = SwzTile<D>;
  using G = FewGeom<D, CB, Q8>;
  constexpr int kRows = G::kRows, kNC = T::kNC, kKS = D / 32, kDB = D / 16;
  constexpr int kLoads = Q8 ? kNC / 2 : kNC;  // of 16 positions: 64 bytes of each
  float2(*const join)[kRows] = reinterpret_cast<float2(*)[kRows]>(smem + kFewWaves * G::kWaveBytes);

  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));  // what depends on it is not kept from item to item, where it goes to scratch
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), m = lane & 15, g = lane >> 4;
  const int rows = w.s.n * a.group, row0 = w.block * kRows, t0 = w.t0;
  const int seen = paged_visible(w.s.keys, w.s.n, (min(rows, row0 + kRows) - 1) / a.group, a.causal);
  const int all_see = paged_visible(w.s.keys, w.s.n, row0 / a.group, a.causal);
  const int units = min(2 * w.t1, (seen + kUnit - 1) / kUnit) - 2 * t0;  // of the part
  const int u0 = 2 * t0 + max(units, 0) * wave / kFewWaves, u1 = 2 * t0 + max(units, 0) * (wave + 1) / kFewWaves;

  // Where 64 stretches of 16 positions lie in the cache, lane l's being stretch from + l; behind the last one it is that one.
  bool bad = w.s.past;
  const int last_stretch = (w.s.keys - 1) >> 4;
  int from = 0;
  long k_at = 0, v_at = 0, ks_at = 0, vs_at = 0;
  auto fetch = [&](int first) __attribute__((always_inline)) {
    from = first;
    const int pos = min(first + lane, last_stretch) * 16, page_at = pos / a.page_size, slot = pos - page_at * (int)a.page_size;
    int id = a.table[w.b * a.table_stride + page_at];
    const bool none = (unsigned)id >= (unsigned)a.pages;
    // of stretches that are behind the wave's last one nothing is said
    bad |= __builtin_amdgcn_ballot_w64(none && first + lane < 2 * u1) != 0;
    if (none) id = 0;
    k_at = id * a.ks.page + (long)slot * a.ks.slot;
    v_at = id * a.vs.page + (long)slot * a.vs.slot;
    if constexpr (Q8) {
      ks_at = id * a.kss.page + (long)slot * a.kss.slot;
      vs_at = id * a.vss.page + (long)slot * a.vss.slot;
    }
  };
  if (u0 < u1) fetch(2 * u0);
  // stretch R of unit u: the lane that has it, and how many positions it has, less one
  auto lane_of = [&](int u, int R) __attribute__((always_inline)) { return min(2 * u + R, last_stretch) - from; };
  auto last_of = [&](int u, int R) __attribute__((always_inline)) { return w.s.keys - 1 - min(2 * u + R, last_stretch) * 16; };

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

  char* const tile = smem + wave * G::kWaveBytes;
  const int r16 = lane >> 2, q4 = lane & 3;
  const char* const k_head = a.k + (long)w.head * a.ks.head;
  const char* const v_head = a.v + (long)w.head * a.vs.head;

  f4v o[CB][kDB];
  float mc[CB], l[CB], mv[CB];  // mv: m' of an 8-bit cache
#pragma unroll
  for (int cb = 0; cb < CB; ++cb) {
    mc[cb] = mv[cb] = -INFINITY, l[cb] = 0.f;
#pragma unroll
    for (int db = 0; db < kDB; ++db) o[cb][db] = f4v{0.f, 0.f, 0.f, 0.f};
  }
  // exponents of the lane's 8 keys: scores times c, without those that its row does not see
  auto exponents = [&](int u, int cb, const f4v (&s)[2], float (&t)[8]) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < 8; ++e) t[e] = s[e >> 2][e & 3] * a.c;
    if (u * kUnit + kUnit > all_see) {
      asm volatile("");  // stays a branch
      const int left = sees[cb] - u * kUnit - 16 * (g >> 1) - 4 * (g & 1);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (8 * (e >> 2) + (e & 3) >= left) t[e] = -INFINITY;
    }
  };
  int odd = u1;  // first unit whose values were not all numbers; those that were none are 0 in its tile
  // the maximum of theirs and all lanes' of the row and m; no key yet is taken as 0: every exponential is 0 then
  auto raise = [&](const float (&t)[8], float& m, float& from) __attribute__((always_inline)) {
    float mx = t[0];
#pragma unroll
    for (int e = 1; e < 8; ++e) mx = fmaxf(mx, t[e]);
    mx = fmaxf(max_over_groups(mx), m);
    from = mx == -INFINITY ? 0.f : mx;
    const float alpha = fast_exp2(m - from);
    m = mx;
    return alpha;
  };

  if constexpr (!Q8) {
    const int col = (q4 ^ swz(r16 >> 2)) * 16;
    char* const v_tile = tile + G::kTileBytes;
    u4v kr[2][kLoads], vr[2][kLoads];
    const int k_lane = r16 * a.ks.slot + col, v_lane = r16 * a.vs.slot + col;
    auto load = [&](int u) __attribute__((always_inline)) {
      if (2 * u - from >= 64) fetch(2 * u);
#pragma unroll
      for (int R = 0; R < 2; ++R) {
        const char* const kb = k_head + of_lane(k_at, lane_of(u, R));
        const char* const vb = v_head + of_lane(v_at, lane_of(u, R));
        int ko = k_lane, vo = v_lane;
        if (last_of(u, R) < 15) {  // positions past the last one: the last one again
          asm volatile("");
          const int past = max(r16 - last_of(u, R), 0);
          ko -= past * a.ks.slot, vo -= past * a.vs.slot;
        }
#pragma unroll
        for (int i = 0; i < kLoads; ++i) kr[R][i] = *reinterpret_cast<const u4v*>(kb + (unsigned)(ko + 64 * i));
#pragma unroll
        for (int i = 0; i < kLoads; ++i) vr[R][i] = *reinterpret_cast<const u4v*>(vb + (unsigned)(vo + 64 * i));
      }
    };
    const unsigned ka0 = opaque_lds_address(tile + rows16_off<D>(lane, 0)), ka1 = opaque_lds_address(tile + rows16_off<D>(lane, 1));
    const Cols16<D> va(v_tile, lane);
    if (u0 < u1) load(u0);
    for (int u = u0; u < u1; ++u) {
#pragma unroll
      for (int R = 0; R < 2; ++R) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
          *reinterpret_cast<u4v*>(tile + T::block_off(R, i) + lane * 16) = kr[R][i];
          *reinterpret_cast<u4v*>(v_tile + T::block_off(R, i) + lane * 16) = vr[R][i];
        }
      }
      if (u + 1 < u1) load(u + 1);
      if (u * kUnit + kUnit > all_see) {
        asm volatile("");
        auto at = [&](int i) __attribute__((always_inline)) { return reinterpret_cast<u4v*>(v_tile + i * 1024 + lane * 16); };
        Finite<BF> finite;
#pragma unroll
        for (int i = 0; i < 2 * kLoads; ++i) finite.look(*at(i));
        if (__builtin_expect(!finite.all(), false)) {
          odd = min(odd, u);
#pragma unroll
          for (int i = 0; i < 2 * kLoads; ++i) *at(i) = Finite<BF>::numbers(*at(i));
        }
      }
      f4v s[CB][2];
      h8 frag[2 * kKS];  // asked for together, and again those of V in front of the exponentials
#pragma unroll
      for (int n = 0; n < 2 * kKS; ++n) frag[n] = rows16_at<D>(ka0, ka1, n & 1, n >> 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int n = 0; n < 2 * kKS; ++n) {
        const int p = n & 1, kk = n >> 1;
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) s[cb][p] = mma16<BF>(frag[n], qf[cb][kk], kk == 0 ? f4v{0.f, 0.f, 0.f, 0.f} : s[cb][p]);
      }
      static_assert(kDB == 2 * kKS, "");
      if (CB == 1) {
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int db = 0; db < kDB; ++db) frag[db] = va.at(0, 0, db);
        __builtin_amdgcn_sched_barrier(0);
      }
      u4v pf[CB];
      float alpha[CB];
      bool moved = false;
#pragma unroll
      for (int cb = 0; cb < CB; ++cb) {
        float t[8], from, sum = 0.f;
        exponents(u, cb, s[cb], t);
        alpha[cb] = raise(t, mc[cb], from);
        moved |= alpha[cb] != 1.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          t[e] = fast_exp2(t[e] - from);
          sum += t[e];
        }
        l[cb] = l[cb] * alpha[cb] + sum;
#pragma unroll
        for (int e = 0; e < 4; ++e) pf[cb][e] = pack2<BF>(t[2 * e], t[2 * e + 1]);
      }
      if (__builtin_amdgcn_ballot_w64(moved)) {
#pragma unroll
        for (int cb = 0; cb < CB; ++cb)
#pragma unroll
          for (int db = 0; db < kDB; ++db) o[cb][db] *= alpha[cb];
      }
#pragma unroll
      for (int db = 0; db < kDB; ++db) {
        const h8 vf = CB == 1 ? frag[db] : va.at(0, 0, db);
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) o[cb][db] = mma16<BF>(vf, __builtin_bit_cast(h8, pf[cb]), o[cb][db]);
      }
    }
  } else {
    typedef __attribute__((address_space(3))) u2v lds_u2v;
    typedef __attribute__((address_space(3))) u4v lds_u4v;
    typedef __attribute__((address_space(3))) unsigned lds_u;
    typedef int i2v __attribute__((ext_vector_type(2)));
    typedef __attribute__((address_space(3))) i2v lds_i2v;
    const unsigned lds0 = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)tile;
    // Chunk c of 16 bytes of row r16 of rows 16 R .. lies at (c ^ swz(r16 >> 2) ^ 2 R) * 16 of the row's 64 bytes, so that neither
    // reads below meet in a bank.
    const int col = (q4 ^ swz(r16 >> 2)) * 16;
    constexpr float kUp = BF ? 0.f : 14.f;  // the largest probability's exponent
    constexpr int kBack = 960 * (kLoads - 1), kOps = 4 * kLoads + 1;  // see copy16_blocks; copies of a unit
    auto copy = [&](const char* from, int off, unsigned to) __attribute__((always_inline)) {
      if constexpr (kLoads == 1) copy16(wave_uniform(from), off, smem + __builtin_amdgcn_readfirstlane(to - lds0) + wave * G::kWaveBytes);
      else copy16_blocks<kLoads>(wave_uniform(from - kBack), off + kBack, __builtin_amdgcn_readfirstlane(to));
    };
    const int k_lane = r16 * a.ks.slot, v_lane = r16 * a.vs.slot;
    // scales of the 32 keys, then of the values, a lane each
    const unsigned char* const sc_head = lane < 32 ? a.k_scale + (long)w.head * a.kss.head : a.v_scale + (long)w.head * a.vss.head;
    const int sc_slot = lane < 32 ? a.kss.slot : a.vss.slot;
    auto ask = [&](int u, unsigned slot) __attribute__((always_inline)) {
      if (2 * u - from >= 64) fetch(2 * u);
      int sc_row = lane & 15;
#pragma unroll
      for (int R = 0; R < 2; ++R) {
        int ko = k_lane + (col ^ (32 * R)), vo = v_lane + (col ^ (32 * R));
        if (last_of(u, R) < 15) {  // positions past the last one: the last one again
          asm volatile("");
          const int past = max(r16 - last_of(u, R), 0);
          ko -= past * a.ks.slot, vo -= past * a.vs.slot;
          if ((lane >> 4 & 1) == R) sc_row = min(sc_row, last_of(u, R));
        }
        copy(k_head + of_lane(k_at, lane_of(u, R)), ko, slot + R * kLoads * 1024);
        copy(v_head + of_lane(v_at, lane_of(u, R)), vo, slot + G::kTileBytes + R * kLoads * 1024);
      }
      const long ks = lane & 16 ? of_lane(ks_at, lane_of(u, 1)) : of_lane(ks_at, lane_of(u, 0));
      const long vs = lane & 16 ? of_lane(vs_at, lane_of(u, 1)) : of_lane(vs_at, lane_of(u, 0));
      copy_byte(sc_head + (lane < 32 ? ks : vs) + (long)sc_row * sc_slot, __builtin_amdgcn_readfirstlane(slot + 2 * G::kTileBytes));
    };
    unsigned k_row[2];  // the lane's row of keys: 8 p + (m & 7) of rows 16 (m >> 3) ..
    unsigned k_scale_at[2], v_scale_at[2];
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const int R = m >> 3, row = 8 * p + (m & 7);
      k_row[p] = lds0 + R * kLoads * 1024 + row * 64 + (((g >> 1) ^ swz(row >> 2) ^ (2 * R)) * 16) + (g & 1) * 8;
      k_scale_at[p] = lds0 + 2 * G::kTileBytes + (16 * R + row) * 4;
      v_scale_at[p] = lds0 + 2 * G::kTileBytes + (32 + 16 * (g >> 1) + 8 * p + 4 * (g & 1)) * 4;
    }
    unsigned v_row;  // of 8 keys of the lane's group, in the order of its probabilities, a pair of lanes has 16 features of each
    {
      const int R = g >> 1, row = 4 * (g & 1) + (m >> 1 & 3) + 8 * (m >> 3);
      v_row = lds0 + G::kTileBytes + R * kLoads * 1024 + row * 64 + ((swz(row >> 2) ^ (2 * R)) * 16) + (m & 1) * 8;
    }
    if (u0 < u1) ask(u0, lds0);
    if (u0 + 1 < u1) ask(u0 + 1, lds0 + G::kSlotBytes);
    for (int u = u0; u < u1; ++u) {
      const unsigned slot = (u - u0) & 1 ? G::kSlotBytes : 0;
      if (u + 1 < u1) wait_vm<kOps>();
      else wait_vm<0>();
      asm volatile("" ::: "memory");
      if (u * kUnit + kUnit > all_see) {  // 0x7f and 0xff are NaN
        asm volatile("");
        auto at = [&](int i) __attribute__((always_inline)) { return (lds_u4v*)(uintptr_t)(lds0 + slot + G::kTileBytes + i * 1024 + lane * 16); };
        auto nan = [](u4v x) __attribute__((always_inline)) { return ((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; };
        u4v any = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 2 * kLoads; ++i) any |= nan(*at(i));
        if (__builtin_expect(__builtin_amdgcn_ballot_w64((any[0] | any[1] | any[2] | any[3]) != 0) != 0, false)) {
          odd = min(odd, u);
#pragma unroll
          for (int i = 0; i < 2 * kLoads; ++i) *at(i) = *at(i) & ~((nan(*at(i)) >> 7) * 0xffu);
        }
      }
      f4v s[CB][2];
      // asked for together: scales, K, and in front of the exponentials V
      float scale[2];
      u4v e4[2];
      u2v frag[2 * kKS];
#pragma unroll
      for (int p = 0; p < 2; ++p) scale[p] = scale_of(*(const lds_u*)(uintptr_t)(k_scale_at[p] + slot));
#pragma unroll
      for (int n = 0; n < 2 * kKS; ++n)
        frag[n] = *(const lds_u2v*)(uintptr_t)(((k_row[n & 1] + slot) ^ (n >> 1 & 1) * 32) + (n >> 2) * 1024);
#pragma unroll
      for (int p = 0; p < 2; ++p) e4[p] = *(const lds_u4v*)(uintptr_t)(v_scale_at[p] + slot);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int n = 0; n < 2 * kKS; ++n) {
        const int p = n & 1, kk = n >> 1;
        const h8 kf = __builtin_bit_cast(h8, from_e4m3<BF>(frag[n][0], frag[n][1], scale[p]));
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) s[cb][p] = mma16<BF>(kf, qf[cb][kk], kk == 0 ? f4v{0.f, 0.f, 0.f, 0.f} : s[cb][p]);
      }
      static_assert(kDB == 2 * kKS, "");
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int db = 0; db < kDB; ++db)
        frag[db] = __builtin_bit_cast(u2v, __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i2v*)(uintptr_t)(((v_row + slot) ^ (db & 3) * 16) + (db >> 2) * 1024)));
      __builtin_amdgcn_sched_barrier(0);
      float e8[8];  // exponents of the lane's values
#pragma unroll
      for (int e = 0; e < 8; ++e) e8[e] = (float)(int)(e4[e >> 2][e & 3] - 127);
      u4v pf[CB];
      float alpha[CB];
      bool moved = false;
#pragma unroll
      for (int cb = 0; cb < CB; ++cb) {
        float t[8], from, sum = 0.f;
        exponents(u, cb, s[cb], t);
        const float less = raise(t, mc[cb], from);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum += fast_exp2(t[e] - from);
        l[cb] = l[cb] * less + sum;
#pragma unroll
        for (int e = 0; e < 8; ++e) t[e] += e8[e];
        alpha[cb] = raise(t, mv[cb], from);
        from -= kUp;
        moved |= alpha[cb] != 1.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) pf[cb][e] = pack2<BF>(fast_exp2(t[2 * e] - from), fast_exp2(t[2 * e + 1] - from));
      }
      if (__builtin_amdgcn_ballot_w64(moved)) {
#pragma unroll
        for (int cb = 0; cb < CB; ++cb)
#pragma unroll
          for (int db = 0; db < kDB; ++db) o[cb][db] *= alpha[cb];
      }
#pragma unroll
      for (int db = 0; db < kDB; ++db) {
        const h8 vf = __builtin_bit_cast(h8, from_e4m3<BF>(frag[db][0], frag[db][1], 1.f));
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) o[cb][db] = mma16<BF>(vf, __builtin_bit_cast(h8, pf[cb]), o[cb][db]);
      }
      staged_rows_read();  // the slot has been read
      if (u + 2 < u1) ask(u + 2, lds0 + slot);
    }
    // back to the scale of the sums: the exponents are at most the largest of the scales apart
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) {
      const float f = mc[cb] == -INFINITY ? 0.f : fast_exp2(mv[cb] - mc[cb] - kUp);
#pragma unroll
      for (int db = 0; db < kDB; ++db) o[cb][db] *= f;
    }
  }

  if (__builtin_expect(odd < u1, false)) {
    for (int key = odd * kUnit; key < min(u1 * kUnit, w.s.keys); ++key) {
      const ValueRow v = value_row<Q8>(a, w, key);
      if (!v.at) continue;
#pragma unroll
      for (int db = 0; db < kDB; ++db) {
        const u2v x = values4<BF, Q8>(v.at, db * 16 + 4 * g, 1.f);
#pragma unroll
        for (int cb = 0; cb < CB; ++cb)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (key < sees[cb]) o[cb][db][r] = Finite<BF>::with_other(o[cb][db][r], x[r >> 1] >> (16 * (r & 1)) & 0xffffu);
      }
    }
  }

  if (a.shared && w.opens && threadIdx.x < kRows && row0 + (int)threadIdx.x < rows) {
    const int row = row0 + threadIdx.x, token = row / a.group, head = w.head * (int)a.group + row - token * (int)a.group;
    a.places[(w.s.first + token) * a.head + head] = int2{paged_first_row(w.stretch, w.parts, slot_rows) + (int)threadIdx.x, w.parts};
  }
  // the waves' sums, relative to the largest maximum
#pragma unroll
  for (int cb = 0; cb < CB; ++cb) {
    const float sum = over_groups_sum(l[cb]);
    if (g == 0) join[wave][16 * cb + m] = float2{mc[cb], bad ? NAN : sum};
  }
  block_barrier();
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
  block_barrier();
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
    if (w.whole) {
      const int token = (row0 + row) / a.group, head = w.head * (int)a.group + (row0 + row - token * a.group);
      const float inv = sum == 0.f ? of_no_score(w, token, a.causal, NAN) : 1.f / sum;
      store4<BF>(a.o + (((long)(w.s.first + token) * a.head + head) * D + piece * 4) * 2, x * inv);
    } else {
      const long at = (long)w.place * slot_rows + row;
      *reinterpret_cast<f4v*>(a.part_o + at * D + piece * 4) = x;
      if (piece == 0) a.part_ml[at] = float2{mx, sum == 0.f ? of_no_score(w, (row0 + row) / a.group, a.causal, 1.f) : sum};
    }
  }
}

// ---------------------------------------------------------------------------
// Attention, blocks of 128 rows.  Work group = 4 waves of 32 rows each, one per SIMD, two work groups to a CU; K and V in tiles of 64
// keys with two slots of LDS each, 16 rows of a tile copied by each wave from one page.  The steps are those of the 128-query
// forward for equal lengths: softmax(j) with the MFMAs of accumulate(j - 1) and scores(j + 1) between its vector
// instructions, the running maximum raised only where a tile's probabilities come out too large: written out here and there, so that a
// mistake in one is to be looked for in the other.  New tokens stand anywhere
// against the tiles, so up to two tiles of a wave need a mask; they are done after the main loop.
//
// Bound by the MFMAs with what stands between them: 4096 new tokens of 32768, 32 heads of 128, fp16 1845 us, 1.12 PFLOP/s of the
// 1.24 that a large library product reaches; 2048 of 16384 475 us, 1.09 (bf16 445, 1.16; 8-bit cache 519, 0.99; heads of 64 290, 0.89).
// With few blocks, by the parts' sums, 64 KiB each, and by the beginnings: 512 of 8192 83 us, 0.80 PFLOP/s, 10 of them for the join.
// ---------------------------------------------------------------------------
template <int D, bool Q8>
struct ManyGeom {
  static constexpr int kPitch = 64 * 4 + 16;  // of a row of 64 sums in LDS
  static constexpr int kTileBytes = 4 * SwzTile<D>::kBytes, kStageBytes = kPagedThreads / 64 * kResident * kPitch;
  static constexpr int kFlags = kTileBytes > kStageBytes ? kTileBytes : kStageBytes;  // where the waves say that a page is bad
  static constexpr int kRaw = 16 * D;  // bytes of 16 rows in 8 bits
  static constexpr int kBytes = Q8 ? kFlags + kPagedThreads / 64 * 2 * kRaw : kFlags + 16;
};
constexpr float kNoMaximum = -3.4028234663852886e38f;  // in the place of -inf: a difference of two of them is 0

template <bool BF>
__device__ __forceinline__ f16v mma32(h8 x, h8 y, f16v z) {
  if constexpr (BF) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, x), __builtin_bit_cast(b8, y), z, 0, 0, 0);
  else return mfma(x, y, z);
}
// pack2 at this place in the program: seen through, the optimiser moves conversions past the next branch.
template <bool BF>
__device__ __forceinline__ unsigned pack2_here(float x, float y) {
  unsigned r = pack2<BF>(x, y);
  asm volatile("" : "+v"(r));
  return r;
}

template <int D, bool BF, bool Q8>
__device__ __forceinline__ void many_rows(const PagedArgs& a, const Part& w, char* smem) {
  using M = ManyGeom<D, Q8>;
  using G = TileGeom<D>;
  using T = SwzTile<D>;
  constexpr int kDB = G::kDBlocks, kIPW = T::kNC;  // copies of a wave and tile: 16 rows, 64 bytes of each
  constexpr int kVOff = 2 * T::kBytes;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // what depends on the lane is worked out again where it is needed, not kept in registers across the main loop
  auto lane_now = []() __attribute__((always_inline)) {
    int t = threadIdx.x;
    asm volatile("" : "+v"(t));
    return t & 63;
  };
  const int rows = w.s.n * a.group, row0 = w.block * kManyRows, row0w = row0 + wave * kResident;
  const int t0 = w.t0, nt = w.t1 - t0;
  int ntw = 0, nfull = 0;  // tiles that the wave works on, those of them that all its rows see whole
  if (row0w < rows) {
    ntw = min(max(paged_tiles(paged_visible(w.s.keys, w.s.n, (min(rows, row0w + kResident) - 1) / a.group, a.causal)) - t0, 0), nt);
    nfull = min(max(paged_visible(w.s.keys, w.s.n, row0w / a.group, a.causal) / kPagedTile - t0, 0), nt);
  }
  const int jm = min(nfull, ntw - 1);  // steps of the main loop, with the first

  // Offsets in the cache of this wave's 16 rows of 64 tiles, lane l those of tile from + l; in the lane's registers.
  const char* const k_head = a.k + (long)w.head * a.ks.head;
  const char* const v_head = a.v + (long)w.head * a.vs.head;
  const int last_stretch = (w.s.keys - 1) >> 4;
  const int k_shift = a.k_shift, v_shift = a.v_shift;
  unsigned k_at = 0, v_at = 0, ks_at = 0, vs_at = 0;
  int at_from = 0;
  bool bad = w.s.past;
  auto fetch_at = [&](int j) __attribute__((always_inline)) {
    at_from = j;
    const PagedArgs a = args_again();
    const int lane = lane_now(), stretch = min(4 * (t0 + j + lane) + wave, last_stretch);
    const int pos = stretch * 16, page_at = pos / a.page_size, slot = pos - page_at * (int)a.page_size;
    int id = a.table[w.b * a.table_stride + page_at];
    const bool none = (unsigned)id >= (unsigned)a.pages;
    bad |= __builtin_amdgcn_ballot_w64(none && j + lane < nt) != 0;
    if (none) id = 0;
    k_at = (unsigned)((id * a.ks.page + (long)slot * a.ks.slot) >> a.k_shift);
    v_at = (unsigned)((id * a.vs.page + (long)slot * a.vs.slot) >> a.v_shift);
    asm volatile("" : "+v"(k_at), "+v"(v_at));
    if constexpr (Q8) {
      ks_at = (unsigned)(id * a.kss.page + (long)slot * a.kss.slot);
      vs_at = (unsigned)(id * a.vss.page + (long)slot * a.vss.slot);
      asm volatile("" : "+v"(ks_at), "+v"(vs_at));
    }
  };
  constexpr int kCopies = Q8 ? kIPW / 2 : kIPW, kBack = 960 * (kCopies - 1);  // see copy16_blocks
  int k_goff, v_goff;
  {
    const int lane = lane_now(), r16 = lane >> 2, col = (Q8 ? lane & 3 : (lane & 3) ^ swz(r16 >> 2)) * 16;
    k_goff = r16 * a.ks.slot + col + kBack;
    v_goff = r16 * a.vs.slot + col + kBack;
    asm volatile("" : "+v"(k_goff), "+v"(v_goff));
  }
  const unsigned lds0 = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)smem;
  const unsigned lds_w = lds0 + wave * (kIPW * 1024);
  auto past_end = [&](int j, int off, bool value) __attribute__((always_inline)) {  // rows behind the last key: that one
    const PagedArgs a = args_again();
    const int stride = value ? a.vs.slot : a.ks.slot;
    const int lane = lane_now(), stretch = min(4 * (t0 + j) + wave, last_stretch);
    const int r16 = lane >> 2;
    return off - max(r16 - (w.s.keys - 1 - stretch * 16), 0) * stride;
  };
  const int j_end = (w.s.keys - 1) / kPagedTile - t0;  // the tile with the last key
  // 64 bytes of 16 rows to each 1 KiB from `to` on
  auto copy = [&](const char* head, unsigned at, int shift, int off, int j, bool value, unsigned to) __attribute__((always_inline)) {
    const char* const from = head + ((long)(unsigned)__builtin_amdgcn_readlane(at, j - at_from) << shift) - kBack;
    if (j == j_end) off = past_end(j, off, value);
    if constexpr (kCopies == 1) copy16(wave_uniform(from), off, smem + __builtin_amdgcn_readfirstlane(to - lds0));
    else copy16_blocks<kCopies>(wave_uniform(from), off, __builtin_amdgcn_readfirstlane(to));
  };
  auto copy_k = [&](int j, unsigned to) __attribute__((always_inline)) { copy(k_head, k_at, k_shift, k_goff, j, false, to); };
  auto copy_v = [&](int j, unsigned to) __attribute__((always_inline)) { copy(v_head, v_at, v_shift, v_goff, j, true, to); };
  // A cache in 8 bits: rows come to LDS as they are, to a place of the wave's own, with their scales in registers, and go from there
  // to the tile a step later.
  const unsigned raw_k = lds0 + M::kFlags + wave * 2 * M::kRaw, raw_v = raw_k + M::kRaw;
  unsigned k_sc = 0, v_sc = 0;
  auto scale_from = [&](const unsigned char* scales, unsigned at, int j, bool value) __attribute__((always_inline)) -> unsigned {
    const PagedArgs a = args_again();
    const CacheStrides st = value ? a.vss : a.kss;
    const int r16 = min(lane_now() >> 2, w.s.keys - 1 - min(4 * (t0 + j) + wave, last_stretch) * 16);
    const unsigned char* const from = scales + (long)w.head * st.head + (unsigned)__builtin_amdgcn_readlane(at, j - at_from);
    return from[(unsigned)(r16 * st.slot)];
  };
  auto ask_k = [&](int j, unsigned to, unsigned& sc) __attribute__((always_inline)) {
    copy_k(j, to);
    sc = scale_from(args_again().k_scale, ks_at, j, false);
  };
  auto ask_v = [&](int j) __attribute__((always_inline)) {
    copy_v(j, raw_v);
    v_sc = scale_from(args_again().v_scale, vs_at, j, true);
  };
  // Of a lane's 16 values one half is chunk c, the other c ^ 1 of a row; lanes two apart write the same banks, so they begin with
  // different halves.
  typedef __attribute__((address_space(3))) u2v lds_u2v;
  typedef __attribute__((address_space(3))) u4v lds_u4v;
  struct Put {
    unsigned from[2], to[2];  // the lane's halves of raw rows of K and its chunks of the first tile, the half that it begins with first
  };
  auto put_lane = [&]() __attribute__((always_inline)) {
    const int lane = lane_now(), r16 = lane >> 2, q4 = lane & 3, first = q4 >> 1;
    Put p;
    p.from[0] = raw_k + lane * 16 + first * 8;
    p.to[0] = lds0 + T::block_off(wave, first) + r16 * 64 + (((2 * (q4 & 1) + first) ^ swz(r16 >> 2)) * 16);
    p.from[1] = p.from[0] ^ 8, p.to[1] = p.to[0] ^ 16;
#pragma unroll
    for (int half = 0; half < 2; ++half) asm volatile("" : "+v"(p.from[half]), "+v"(p.to[half]));
    return p;
  };
  auto put_from = [&](const Put& p, bool value, int i, int half) __attribute__((always_inline)) {
    return *(const lds_u2v*)(uintptr_t)(p.from[half] + (value ? M::kRaw : 0) + 1024 * i);
  };
  auto put_to = [&](const Put& p, unsigned tile, u2v x, float scale, int i, int half) __attribute__((always_inline)) {
    *(lds_u4v*)(uintptr_t)(p.to[half] + tile + T::block_off(0, 2 * i)) = from_e4m3<BF>(x[0], x[1], scale);
  };
  auto put = [&](bool value, unsigned sc, unsigned tile) __attribute__((always_inline)) {
    const Put p = put_lane();
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
      const u2v x = put_from(p, value, i, 0), y = put_from(p, value, i, 1);
      put_to(p, tile, x, scale_of(sc), i, 0);
      put_to(p, tile, y, scale_of(sc), i, 1);
    }
  };

  if (nt > 0) fetch_at(0);
  // All that comes from memory first is asked for together: pages, rows of q, then K.  The rows of q go through the slots of V, which
  // comes later.
  char* const my_rows = smem + kVOff + wave * (T::kBytes / 2);
  u4v q_rows[2][T::kNC];
  {
    const int lane = lane_now(), r16 = lane >> 2, col = ((lane & 3) ^ swz(r16 >> 2)) * 16;
    const char* const base = a.q + w.b * a.q_batch + (a.ends ? w.s.first : 0) * a.q_seq + (long)w.head * (int)a.group * a.q_head;
#pragma unroll
    for (int R = 0; R < 2; ++R) {
      const int row = min(row0w + 16 * R + r16, rows - 1), token = row / a.group;
      const char* const from = base + token * a.q_seq + (row - token * (int)a.group) * a.q_head + col;
#pragma unroll
      for (int C = 0; C < T::kNC; ++C) q_rows[R][C] = *reinterpret_cast<const u4v*>(from + C * 64);
    }
  }
  if (nt > 0) {
    if constexpr (Q8) {
      unsigned k_sc1 = 0;
      ask_k(0, raw_k, k_sc);
      if (nt > 1) ask_k(1, raw_v, k_sc1);
      wait_vm<0>();
      asm volatile("" ::: "memory");
      put(false, k_sc, 0);
      if (nt > 1) put(true, k_sc1, T::kBytes);
      staged_rows_read();
      if (nt > 2) ask_k(2, raw_k, k_sc);
      ask_v(0);
    } else {
      copy_k(0, lds_w);
      if (nt > 1) copy_k(1, lds_w + T::kBytes);
    }
  }
#pragma unroll
  for (int R = 0; R < 2; ++R)
#pragma unroll
    for (int C = 0; C < T::kNC; ++C) *reinterpret_cast<u4v*>(my_rows + T::block_off(R, C) + lane_now() * 16) = q_rows[R][C];
  h8 qf[G::kKSteps];
  {
    const StagedRows<D> staged{my_rows, lane_now()};
    staged_rows_read();
#pragma unroll
    for (int kk = 0; kk < G::kKSteps; ++kk) qf[kk] = staged.wide(kk);
    staged_rows_read();
  }
  if (!(a.c > 0.f)) {  // the maximum of scores times c is c times their maximum only for c > 0
#pragma unroll
    for (int kk = 0; kk < G::kKSteps; ++kk) {
      qf[kk] = a.c < 0.f ? -qf[kk] : h8{};
      asm volatile("" : "+v"(qf[kk]));
    }
  }
  const float c = a.c == 0.f ? 1.f : fabsf(a.c);
  int k_off[2], v_off[2];
  swz_rows_off<D>(lane_now(), k_off);
  swz_cols_off<D>(lane_now(), v_off);
  const unsigned ka0 = opaque_lds_address(smem + k_off[0]), ka1 = opaque_lds_address(smem + k_off[1]);
  const unsigned va0 = opaque_lds_address(smem + v_off[0]), va1 = opaque_lds_address(smem + v_off[1]);
  auto k_frag = [&](unsigned at, int n) __attribute__((always_inline)) { return swz_rows_at<D>(ka0 + at, ka1 + at, n & 1, n >> 1); };
  auto v_frag = [&](unsigned at, int n) __attribute__((always_inline)) {
    return swz_cols_at<D>(va0 + kVOff + at, va1 + kVOff + at, n / kDB, n % kDB);
  };

  f16v o[kDB], zero;
#pragma unroll
  for (int r = 0; r < 16; ++r) zero[r] = 0.f;
#pragma unroll
  for (int db = 0; db < kDB; ++db) o[db] = zero;
  float mc = kNoMaximum, l_run = 0.f;
  f16v sA[2], sB[2];
  u4v pf[4];  // probabilities of a tile, pairs of 16 bits in B-operand order

  constexpr int kLead = 3;  // LDS fragments are read this many MFMAs ahead
  constexpr int kNS = 2 * G::kKSteps, kNP = 4 * kDB;
  auto scores = [&](unsigned at, f16v (&s)[2]) __attribute__((always_inline)) {
    h8 frag[kLead];
#pragma unroll
    for (int n = 0; n < kLead; ++n) frag[n] = k_frag(at, n);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int n = 0; n < kNS; ++n) {
      const int rb = n & 1, kk = n >> 1;
      s[rb] = mma32<BF>(frag[n % kLead], qf[kk], kk == 0 ? zero : s[rb]);
      if (n + kLead < kNS) frag[n % kLead] = k_frag(at, n + kLead);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto exponentials = [&](const f16v (&s)[2]) __attribute__((always_inline)) {
    float l0 = 0.f, l1 = 0.f;
#pragma unroll
    for (int c16 = 0; c16 < 4; ++c16) {
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const float p0 = fast_exp2(fmaf(s[c16 >> 1][(c16 & 1) * 8 + e], c, -mc));
        const float p1 = fast_exp2(fmaf(s[c16 >> 1][(c16 & 1) * 8 + e + 1], c, -mc));
        pf[c16][e >> 1] = pack2_here<BF>(p0, p1);
        l0 += p0;
        l1 += p1;
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    return l0 + l1;
  };
  auto mask = [&](f16v (&s)[2], int j) __attribute__((always_inline)) {
    const PagedArgs a = args_again();
    const int lane = lane_now(), token = min(row0w + (lane & 31), rows - 1) / a.group;
    const int left = paged_visible(w.s.keys, w.s.n, token, a.causal) - (t0 + j) * kPagedTile - 4 * (lane >> 5);
#pragma unroll
    for (int rb = 0; rb < 2; ++rb)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (acc_row(rb, r, 0) >= left) s[rb][r] = -INFINITY;
  };
  auto too_large = [&](float lt) __attribute__((always_inline)) { return __builtin_amdgcn_ballot_w64(!(lt <= 4096.f)) != 0; };
  // probabilities of a tile with the running maximum brought up to date
  auto raise_max = [&](const f16v (&s)[2]) __attribute__((always_inline)) {
    float mx = s[0][0];
#pragma unroll
    for (int rb = 0; rb < 2; ++rb)
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[rb][r]);
    mx = fmaxf(mx, other_half(mx));
    const float mc_new = fmaxf(mc, mx * c);
    const float alpha = fast_exp2(mc - mc_new);
    mc = mc_new;
    l_run *= alpha;
#pragma unroll
    for (int db = 0; db < kDB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[db][r] *= alpha;
    l_run += exponentials(s);
  };
  auto accumulate = [&](unsigned at) __attribute__((always_inline)) {
    h8 frag[kLead];
#pragma unroll
    for (int n = 0; n < kLead; ++n) frag[n] = v_frag(at, n);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int n = 0; n < kNP; ++n) {
      o[n % kDB] = mma32<BF>(frag[n % kLead], __builtin_bit_cast(h8, pf[n / kDB]), o[n % kDB]);
      if (n + kLead < kNP) frag[n % kLead] = v_frag(at, n + kLead);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  int odd = ntw;  // first tile of which only the numbers were multiplied
  auto all_finite = [&](unsigned at) __attribute__((always_inline)) {
    Finite<BF> finite;
#pragma unroll
    for (int n = 0; n < kNP; ++n) {
      finite.look(__builtin_bit_cast(u4v, v_frag(at, n)));
      if (n % 8 == 7) __builtin_amdgcn_sched_barrier(0);
    }
    return finite.all();
  };
  auto accumulate_numbers = [&](unsigned at) __attribute__((always_inline)) {
#pragma unroll
    for (int n = 0; n < kNP; ++n) {
      const h8 v = __builtin_bit_cast(h8, Finite<BF>::numbers(__builtin_bit_cast(u4v, v_frag(at, n))));
      o[n % kDB] = mma32<BF>(v, __builtin_bit_cast(h8, pf[n / kDB]), o[n % kDB]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // Step j uses K(j + 1) and V(j - 1), both in slot (j + 1) & 1; K(j + 2) and V(j) are copied into the other one.  Out of 8 bits
  // they go there now, and K(j + 3) and V(j + 1) are asked for.
  auto top_wait = [&]() __attribute__((always_inline)) {
    wait_vm<0>();
    block_barrier();
  };
  auto fetch_for = [&](int j) __attribute__((always_inline)) {  // the registers hold tiles at_from .. at_from + 63
    if (j + (Q8 ? 3 : 2) - at_from >= 64 && j < nt) fetch_at(j);
  };
  auto next_k = [&](int j, int slot) __attribute__((always_inline)) {
    if constexpr (Q8) {
      if (j + 2 < nt) put(false, k_sc, slot * T::kBytes);
    } else {
      if (j + 2 < nt) copy_k(j + 2, lds_w + slot * T::kBytes);
    }
  };
  auto next_v = [&](int j, int slot) __attribute__((always_inline)) {
    if constexpr (Q8) put(true, v_sc, kVOff + slot * T::kBytes);
    else copy_v(j, lds_w + kVOff + slot * T::kBytes);
  };
  auto ask = [&](int j) __attribute__((always_inline)) {
    if constexpr (Q8) {
      staged_rows_read();  // what lies there has been read
      if (j + 3 < nt) ask_k(j + 3, raw_k, k_sc);
      if (j + 1 < nt) ask_v(j + 1);
    }
  };
  auto top_copy = [&](int j, int slot) __attribute__((always_inline)) {
    fetch_for(j);
    next_k(j, slot);
    if (j < nt) next_v(j, slot);
    ask(j);
  };
  auto step = [&](int j, auto slot_tag, const f16v (&s)[2], f16v (&sn)[2]) __attribute__((always_inline)) {
    constexpr int kSlot = decltype(slot_tag)::value;  // (j + 1) & 1
    constexpr unsigned at = kSlot * T::kBytes;
    constexpr int kM = kNS + kNP;
    h8 frag[kLead];
    u2v raw[Q8 ? 2 * kCopies : 1];
    Put where;
    if constexpr (Q8) where = put_lane();
    float l0 = 0.f, l1 = 0.f, p0 = 0.f, p1 = 0.f;
    auto read = [&](int m) __attribute__((always_inline)) {
      const int ch = m / (2 * kDB), in = m % (2 * kDB);
      return in < kDB ? v_frag(at, ch * kDB + in) : k_frag(at, ch * kDB + in - kDB);
    };
    auto reads = [](int m) { return m >= kM ? 0 : m % (2 * kDB) < kDB ? 2 : 1; };  // LDS reads of a fragment
    auto start = [&](int x) __attribute__((always_inline)) {
      const int c16 = x >> 2, e = (x & 3) * 2;
      p0 = fast_exp2(fmaf(s[c16 >> 1][(c16 & 1) * 8 + e], c, -mc));
      p1 = fast_exp2(fmaf(s[c16 >> 1][(c16 & 1) * 8 + e + 1], c, -mc));
    };
    auto finish = [&](int x) __attribute__((always_inline)) {
      const int c16 = x >> 2, e = (x & 3) * 2;
      l0 += p0;
      l1 += p1;
      asm volatile("" : "+v"(l0), "+v"(l1));  // sums now, not all at the end
      pf[c16][e >> 1] = pack2_here<BF>(p0, p1);
    };
    top_wait();
    fetch_for(j);
#pragma unroll
    for (int m = 0; m < kLead; ++m) frag[m] = read(m);
    constexpr int kCopyKAt = Q8 ? -1 : D == 128 ? 8 : 0;  // K's copies follow when V's are through
    if (!Q8) next_v(j, 1 - kSlot);
    if (kCopyKAt == 0) next_k(j, 1 - kSlot);
    __builtin_amdgcn_sched_barrier(0);
    static_for<kM + 2>([&](auto m_tag) __attribute__((always_inline)) {
      constexpr int m = decltype(m_tag)::value;
      if (kCopyKAt != 0 && m == kCopyKAt) next_k(j, 1 - kSlot);
      if constexpr (Q8) {  // V's halves of 16 rows, then K's, one with every unit; the next are asked for as soon as these are read
        constexpr int kHalves = 2 * kCopies;
        constexpr int kVFirst = 2, kVEnd = kVFirst + kHalves, kKFirst = kVEnd + 2, kKEnd = kKFirst + kHalves;
        if constexpr (m == 0 || m == kVEnd) {
#pragma unroll
          for (int n = 0; n < kHalves; ++n) raw[n] = put_from(where, m == 0, n / 2, n % 2);
        }
        if constexpr (m >= kVFirst && m < kVEnd) {
          constexpr int h = m - kVFirst;
          put_to(where, kVOff + (1 - kSlot) * T::kBytes, raw[h], scale_of(v_sc), h / 2, h % 2);
        }
        if constexpr (m >= kKFirst && m < kKEnd) {
          constexpr int h = m - kKFirst;
          put_to(where, (1 - kSlot) * T::kBytes, raw[h], scale_of(k_sc), h / 2, h % 2);
        }
        if constexpr (m == kKEnd) {
          if (j + 3 < nt) ask_k(j + 3, raw_k, k_sc);
          if (j + 1 < nt) ask_v(j + 1);
        }
      }
      if (m < kM && m % 2 == 0) {  // one wait for the fragments of this unit and the next
        if (D == 64) wait_lds_pinned(reads(m + 2));
        else wait_lds(reads(m + 2));
      }
      if constexpr (m < kM) {
        constexpr int ch = m / (2 * kDB), in = m % (2 * kDB);
        if constexpr (in < kDB) {
          o[in] = mma32<BF>(frag[m % kLead], __builtin_bit_cast(h8, pf[ch]), o[in]);
        } else {
          constexpr int n = ch * kDB + in - kDB, rb = n & 1, kk = n >> 1;
          sn[rb] = mma32<BF>(frag[m % kLead], qf[kk], kk == 0 ? zero : sn[rb]);
        }
        if (m + kLead < kM) frag[m % kLead] = read(m + kLead);
      }
      if (D == 64) {
        if (m >= 1 && m - 1 < 16) finish(m - 1);
        if (m < 16) start(m);
      } else {
        if (m & 1) {
          if (m >= 3 && m < 35) finish((m - 3) / 2);
        } else if (m >= 2 && m < 34) {
          start((m - 2) / 2);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    });
    return l0 + l1;
  };

  if (!Q8) {
    if (nt > 1) wait_vm<kIPW>();  // the second tile of K may still be on its way
    else wait_vm<0>();
  }
  block_barrier();
  if (ntw > 0) scores(0, sA);
  else asm volatile("" : "=v"(sA[0]), "=v"(sA[1]));  // anything: else the compiler keeps 32 zeros for them, in scratch, from item to item
  int j = 0;
  if (jm > 0) {
    top_wait();
    top_copy(0, 0);
    scores(T::kBytes, sB);
    raise_max(sA);
    ++j;
#pragma unroll
    for (int rb = 0; rb < 2; ++rb) sA[rb] = sB[rb];
    // two tiles per round, the scores alternating between two sets of registers
    bool odd_done = false;
    for (;;) {
      int why;
      for (;;) {
        if (!odd_done) {
          if (j >= jm) { why = 0; break; }
          const float lt = step(j, IntTag<0>{}, sA, sB);
          if (too_large(lt)) { why = 1; break; }
          l_run += lt;
          ++j;
        }
        odd_done = false;
        if (j >= jm) { why = 2; break; }
        const float lt = step(j, IntTag<1>{}, sB, sA);
        if (too_large(lt)) { why = 3; break; }
        l_run += lt;
        ++j;
      }
      if (why == 0) break;
      if (why == 2) {
#pragma unroll
        for (int rb = 0; rb < 2; ++rb) sA[rb] = sB[rb];
        break;
      }
      if (why == 1) raise_max(sA);
      else raise_max(sB);
      ++j;
      odd_done = why == 1;
    }
  }
  // the wave's last tiles (up to two with a mask) and the accumulation after them; it goes on copying for the others
  for (; j <= nt; ++j) {
    const unsigned at = ((j + 1) & 1) * T::kBytes;
    top_wait();
    top_copy(j, j & 1);
    if (j > 0 && j <= ntw) {
      if (__builtin_expect(j > nfull && !all_finite(at), false)) {
        odd = min(odd, j - 1);
        accumulate_numbers(at);
      } else {
        accumulate(at);
      }
    }
    if (j < ntw) {
      mask(sA, j);
      raise_max(sA);
      if (j + 1 < ntw) scores(at, sA);
    }
  }

  if (__builtin_expect(odd < ntw, false)) {
    const PagedArgs a = args_again();
    const int lane = lane_now(), token = min(row0w + (lane & 31), rows - 1) / a.group;
    const int sees = paged_visible(w.s.keys, w.s.n, token, a.causal);
    for (int key = (t0 + odd) * kPagedTile; key < min((t0 + ntw) * kPagedTile, w.s.keys); ++key) {
      const ValueRow v = value_row<Q8>(a, w, key);
      if (!v.at) continue;
#pragma unroll
      for (int db = 0; db < kDB; ++db)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const u2v x = values4<BF, Q8>(v.at, db * 32 + 8 * e + 4 * (lane >> 5), v.scale);
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (key < sees) o[db][4 * e + r] = Finite<BF>::with_other(o[db][4 * e + r], x[r >> 1] >> (16 * (r & 1)) & 0xffffu);
        }
    }
  }
  int* const bad_pages = reinterpret_cast<int*>(smem + M::kFlags);
  bad_pages[wave] = bad;  // each wave has looked at a quarter of the pages
  block_barrier();        // every wave is done with the rings: they become the staging tiles
  const PagedArgs z = args_again();
  const int lane = lane_now();
  float l_tot = l_run + other_half(l_run);
  if (bad_pages[0] | bad_pages[1] | bad_pages[2] | bad_pages[3]) l_tot = NAN;
  const int my_token = min(row0w + (lane & 31), rows - 1) / z.group;
  const float none = l_tot == 0.f ? of_no_score(w, my_token, z.causal, w.whole ? NAN : 1.f) : 0.f;
  const float f = !w.whole ? 1.f : l_tot == 0.f ? none : 1.f / l_tot;
  char* const stage = smem + wave * (kResident * M::kPitch);
  const long slot0 = (long)w.place * kManyRows + wave * kResident;
  if (z.shared && w.opens && lane < kResident && row0w + lane < rows) {
    const int row = row0w + lane, token = row / z.group, head = w.head * (int)z.group + row - token * (int)z.group;
    z.places[(w.s.first + token) * z.head + head] = int2{paged_first_row(w.stretch, w.parts, kManyRows) + wave * kResident + lane, w.parts};
  }
  if (!w.whole && lane < kResident && row0w + lane < rows) z.part_ml[slot0 + lane] = l_tot == 0.f ? float2{-INFINITY, none} : float2{mc, l_tot};
#pragma unroll
  for (int half = 0; half < D / 64; ++half) {
#pragma unroll
    for (int db = 0; db < 2; ++db)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        f4v x;
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] = o[2 * half + db][4 * e + r] * f;
        *reinterpret_cast<f4v*>(stage + (lane & 31) * M::kPitch + (db * 32 + 8 * e + 4 * (lane >> 5)) * 4) = x;
      }
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): the wave's own writes have landed
    asm volatile("" ::: "memory");
#pragma unroll
    for (int pass = 0; pass < kResident / 4; ++pass) {
      const int r = 4 * pass + (lane >> 4), row = row0w + r, piece = lane & 15;
      const f4v x = *reinterpret_cast<const f4v*>(stage + r * M::kPitch + piece * 16);
      if (row < rows) {
        if (!w.whole) {
          *reinterpret_cast<f4v*>(z.part_o + (slot0 + r) * D + half * 64 + piece * 4) = x;
        } else {
          const int token = row / z.group, head = w.head * (int)z.group + row - token * (int)z.group;
          store4<BF>(z.o + (((long)(w.s.first + token) * z.head + head) * D + half * 64 + piece * 4) * 2, x);
        }
      }
    }
    __builtin_amdgcn_s_waitcnt(0xC07F);
    asm volatile("" ::: "memory");
  }
}

// ---------------------------------------------------------------------------
// A work group's part, by whichever of the two ways its sequence goes.
// ---------------------------------------------------------------------------
template <int D, int FEW, bool MANY, bool BF, bool Q8>
__global__ void __launch_bounds__(kPagedThreads, 2) paged_forward_kernel(PagedArgs args) {
  using B = Blocks<FEW, MANY, Q8>;
  constexpr int kFewBytes = FEW ? kFewWaves * (FewGeom<D, FEW ? FEW / 16 : 1, Q8>::kWaveBytes + FEW * (int)sizeof(float2)) : 0;
  constexpr int kManyBytes = MANY ? ManyGeom<D, Q8>::kBytes : 0;
  __shared__ __attribute__((aligned(1024))) char smem[kFewBytes > kManyBytes ? kFewBytes : kManyBytes];
  const PagedArgs& a = args;
  if (a.zero_rest) {  // in front of the first sequence and behind the last
    const int first = min(max(a.ends[-1], 0), a.tokens), rest = min(max(a.ends[a.batch - 1], 0), a.tokens);
    const long row = (long)a.head * D * 2, skip = max(rest - first, 0) * row, to = a.tokens * row - skip;
    for (long i = ((long)blockIdx.x * blockDim.x + threadIdx.x) * 16; i < to; i += (long)gridDim.x * blockDim.x * 16)
      *reinterpret_cast<u4v*>(a.o + (i < first * row ? i : i + skip)) = u4v{0, 0, 0, 0};
  }
  touch_args();
  const int lane = threadIdx.x & 63;
  Walk<B> walk;
  if (!walk.begin(a, blockIdx.x, lane)) return;
  for (;;) {
    const PagedArgs a = args_again();
    Part w;
    if (!walk.next(a, lane, w)) return;
    if (MANY && B::many(w.s.n * a.group)) {
      if constexpr (MANY) many_rows<D, BF, Q8>(a, w, smem);
    } else {
      if constexpr (FEW != 0) few_rows<D, FEW / 16, BF, Q8>(a, w, smem, B::kMost);
    }
    if (!walk.more()) return;
    block_barrier();  // the next item takes the same LDS
  }
}

// ---------------------------------------------------------------------------
// Rows whose keys went to several parts.  A slice of D / 4 threads adds up parts of a row, each relative to the largest maximum so
// far.  A work group has one row, whose parts its slices share, or one for each slice; of those with many parts it then takes
// one after the other.  Bound by being a launch of its own where there is little to join (4 us), by its reads of 64 KiB a part of
// many rows otherwise (512 parts 10 us, 3.4 TB/s).
// ---------------------------------------------------------------------------
constexpr int kJoinAhead = 8;  // parts that a slice asks for at a time
struct Joined {
  float m, l;
  f4v x;
};
// A part whose maximum is -inf has sums of 0, and 1 in the place of l if the row sees keys.
__device__ __forceinline__ void join_in(Joined& r, float m, float l, f4v x, float mx) {
  const float f = m == -INFINITY ? 0.f : fast_exp2(m - mx);
  r.l += l * (mx == -INFINITY ? 1.f : f);  // NaN from a bad page stays
  r.x += x * f;
}
template <int D>
__device__ __forceinline__ Joined join_parts(const PagedArgs& a, int at, int parts, int first, int step, int slot_rows, int piece) {
  Joined r{-INFINITY, 0.f, f4v{0.f, 0.f, 0.f, 0.f}};
  for (int p = first; p < parts; p += kJoinAhead * step) {
    float2 ml[kJoinAhead];
    f4v x[kJoinAhead];
#pragma unroll
    for (int u = 0; u < kJoinAhead; ++u) {
      const long row = at + (long)paged_place(0, min(p + u * step, parts - 1)) * slot_rows;
      ml[u] = a.part_ml[row];
      x[u] = *reinterpret_cast<const f4v*>(a.part_o + row * D + piece * 4);
    }
    float mx = r.m;
#pragma unroll
    for (int u = 0; u < kJoinAhead; ++u)
      if (p + u * step < parts) mx = fmaxf(mx, ml[u].x);
    const float f = r.m == -INFINITY ? 0.f : fast_exp2(r.m - mx);
    r.m = mx, r.l *= f, r.x *= f;
#pragma unroll
    for (int u = 0; u < kJoinAhead; ++u)
      if (p + u * step < parts) join_in(r, ml[u].x, ml[u].y, x[u], mx);
  }
  return r;
}

template <int D, bool BF>
__global__ void __launch_bounds__(256) paged_join_kernel(PagedArgs a, int slot_rows, int rows_of_group) {
  constexpr int kPieces = D / 4, kSlices = 256 / kPieces;
  __shared__ Joined sums[kSlices][kPieces];
  const int slice = threadIdx.x / kPieces, piece = threadIdx.x % kPieces, rows = a.tokens * a.head;
  auto place = [&](int row) __attribute__((always_inline)) {
    if (row >= rows) return int2{0, 1};
    if (a.ends) {
      const int token = row / a.head;
      if (token < a.ends[-1] || token >= a.ends[a.batch - 1]) return int2{0, 1};
    }
    int2 r = a.places[row];
    // of tokens that ranges which make no sense left out it says anything
    if (!paged_parts_fit(r.x, r.y, slot_rows)) r.y = 1;
    return r;
  };
  auto store = [&](int row, const Joined& r) __attribute__((always_inline)) {
    store4<BF>(a.o + ((long)row * D + piece * 4) * 2, r.x * (r.l == 0.f ? 0.f : r.m == -INFINITY ? NAN : 1.f / r.l));
  };
  const int row0 = blockIdx.x * rows_of_group;
  if (rows_of_group > 1) {
    const int most = (int)threadIdx.x < rows_of_group ? place(row0 + threadIdx.x).y : 1;
    if (!__syncthreads_or(most > 1)) return;
    if (!__syncthreads_or(most > 2 * kJoinAhead)) {
      for (int u = slice; u < rows_of_group; u += kSlices) {
        const int2 at = place(row0 + u);
        if (at.y > 1) store(row0 + u, join_parts<D>(a, at.x, at.y, 0, 1, slot_rows, piece));
      }
      return;
    }
  }
  for (int u = 0; u < rows_of_group; ++u) {
    const int2 at = place(row0 + u);
    if (at.y == 1) continue;
    __syncthreads();
    sums[slice][piece] = join_parts<D>(a, at.x, at.y, slice, kSlices, slot_rows, piece);
    __syncthreads();
    if (slice) continue;
    float mx = -INFINITY;
#pragma unroll
    for (int v = 0; v < kSlices; ++v) mx = fmaxf(mx, sums[v][piece].m);
    Joined r{mx, 0.f, f4v{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int v = 0; v < kSlices; ++v) join_in(r, sums[v][piece].m, sums[v][piece].l, sums[v][piece].x, mx);
    store(row0 + u, r);
  }
}

// ---------------------------------------------------------------------------
// Writing: a wave to a token, its lanes over 16 bytes of all key heads' keys, then values.  Bound by its bytes: 24576 tokens of 8 key
// heads of 128 into 8 bits 21.8 us, 4.5 TB/s of 5.0 that a copy reaches (asking for all of a token before its place is known 22.8); 64
// tokens 3.3 us, less than the call takes on the host.
// ---------------------------------------------------------------------------
struct WriteArgs {
  const char *k, *v;
  long k_batch, k_seq, k_head, v_batch, v_seq, v_head;  // bytes
  char *kc, *vc;
  unsigned char *k_scale, *v_scale;
  CacheStrides ks, vs, kss, vss;
  const int *table, *keys, *ends;
  long table_stride;
  int batch, tokens, kv_head, pages, width;
  FmhaDivisor page_size, per_sequence;  // per_sequence: new tokens of each, where ends is null
};

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
// Reading: 16 bytes of the result to a lane and step.  Bound by its bytes: 4 x 8192 positions of 8 key heads of 128 out of 8 bits
// 39 us, 4.9 TB/s of 5.0; 1500 of 12 of 64 3.5 us, less than the call takes.  One row after the other 43.5 and 5.3.
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
constexpr int kReadSteps = 4;  // all of whose page numbers are asked for, then all rows

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
  const int row0 = block * (256 * kReadSteps / kChunks) + threadIdx.x / kChunks, chunk = threadIdx.x % kChunks;
  const int* const table = a.table + b * a.table_stride;
  int pos[kReadSteps], head[kReadSteps], slot[kReadSteps], id[kReadSteps];
#pragma unroll
  for (int u = 0; u < kReadSteps; ++u) {
    const int row = row0 + u * (256 / kChunks);
    pos[u] = row / a.kv_head, head[u] = row - pos[u] * (int)a.kv_head;
    const int page_at = pos[u] / a.page_size;
    slot[u] = pos[u] - page_at * (int)a.page_size;
    id[u] = page_at < a.width ? table[page_at] : -1;
  }
  u4v x[kReadSteps];
#pragma unroll
  for (int u = 0; u < kReadSteps; ++u) {
    x[u] = u4v{0, 0, 0, 0};
    if (pos[u] >= min(keys, a.max_seqlen)) continue;
    if (id[u] < 0 || id[u] >= a.pages) {
      x[u] = BF ? u4v{0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u} : u4v{0x7e007e00u, 0x7e007e00u, 0x7e007e00u, 0x7e007e00u};  // NaN
      continue;
    }
    const char* const from = cache + id[u] * st.page + (long)slot[u] * st.slot + (long)head[u] * st.head;
    if constexpr (Q8) {
      const u2v y = *reinterpret_cast<const u2v*>(from + chunk * 8);
      const unsigned s = scales[id[u] * sst.page + (long)slot[u] * sst.slot + (long)head[u] * sst.head];
      x[u] = u4v{y[0], y[1], s, 1};
    } else {
      x[u] = *reinterpret_cast<const u4v*>(from + chunk * 16);
    }
  }
#pragma unroll
  for (int u = 0; u < kReadSteps; ++u) {
    if (pos[u] >= a.max_seqlen) continue;
    if (Q8 && x[u][3] == 1) x[u] = from_e4m3<BF>(x[u][0], x[u][1], scale_of(x[u][2]));  // neither zeros nor NaN end in 1
    *reinterpret_cast<u4v*>(out + (long)(row0 + u * (256 / kChunks)) * (D * 2) + chunk * 16) = x[u];
  }
}

// ---------------------------------------------------------------------------
// Host.
// ---------------------------------------------------------------------------
template <typename... Args>
hipError_t launch(void (*kernel)(Args...), dim3 grid, unsigned block, hipStream_t stream, Args... args) {
  void* ptrs[] = {&args...};
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

struct Launch {
  int few;     // rows of a block of few, 0: there is none
  bool many;   // whether there are blocks of kManyRows
  long items;  // at most
  bool shared;
  int place_rows() const { return many ? kManyRows : few; }
  long grid() const { return shared ? kPagedGroups : (items + 7) / 8 * 8; }
  // Rows that a work group of the second launch looks at: one where most of them have parts, more where few do, as only
  // 2 * kPagedGroups blocks can have any.  Both launches for single tokens of 1000 keys, 32 heads of 128, one row and 32 of them:
  // 160 sequences 106.9 us and 106.5, 256 164.9 and 161.5, 512 312.6 and 305.0, 1024 616 and 601.
  int join_rows(long rows) const { return many || rows > 4096 ? 32 : 1; }
  long join_grid(long rows) const { return (rows + join_rows(rows) - 1) / join_rows(rows); }
};
constexpr long kMostGroups = (1l << 32) / 256 - 1;  // a launch has fewer than 2^32 work items
// The bits below which all offsets of 16 positions are 0, and whether the bits above fit 32.
bool fits(const paged_mha_cache* c, const paged_mha_strides& s, int bytes, int& shift) {
  const unsigned long long page = s.page * bytes, slot = s.slot * bytes * 16, any = page | slot;
  shift = any ? std::min(__builtin_ctzll(any), 31) : 4;
  return ((page * (c->pages - 1) + slot * (c->page_size / 16)) >> shift) < (1ull << 32);
}
Launch plan(const paged_mha_cache* c, const paged_mha_batch* b, int head, int max_new) {
  const long group = head / c->kv_head;
  const long most = (b->cu_seqlens && max_new > 0 ? std::min(max_new, b->tokens) : b->tokens) * group;
  const bool q8 = c->cache_type == PAGED_MHA_E4M3;
  int shift;
  auto all_fit = [&](const paged_mha_strides& s) { return fits(c, s, q8 ? 1 : 2, shift); };
  auto scales_fit = [&](const paged_mha_strides& s) { return s.page * (c->pages - 1) + s.slot * c->page_size < (1LL << 32); };
  Launch p;
  p.many = most > kFewRows && all_fit(c->key_strides) && all_fit(c->value_strides) &&
           (!q8 || (scales_fit(c->key_scale_strides) && scales_fit(c->value_scale_strides)));
  p.few = most <= 16 ? 16 : !p.many || b->cu_seqlens ? kFewRows : 0;
  const int least_rows = p.few ? p.few : kManyRows;
  const long blocks = b->cu_seqlens ? b->tokens * group / least_rows + b->batch : b->batch * ((b->tokens * group + least_rows - 1) / least_rows);
  p.items = blocks * c->kv_head;
  // Items of up to 256 keys are not split: a work group each, unless each would look through a long batch for its own.  us so and shared:
  // 64 sequences of up to 64 keys, 8 key heads 6.5, 11.3; of 200 12.2, 15.4; 200 of 200 26.9, 32.3.
  p.shared = (long)b->table_width * c->page_size * 4 > kPagedLeast || (b->cu_seqlens && b->batch > 64);
  return p;
}
// Sums of the parts' rows, their maxima and totals, where each row of o has its parts.
size_t workspace_bytes_of(const Launch& p, int d, long rows) {
  return p.shared ? (size_t)2 * kPagedGroups * p.place_rows() * (d * 4 + 8) + (size_t)rows * 8 : 0;
}

template <int D, int FEW, bool MANY, bool BF, bool Q8>
int launch_forward(const Launch& p, const PagedArgs& a, hipStream_t stream) {
  if (launch(paged_forward_kernel<D, FEW, MANY, BF, Q8>, dim3(p.grid()), kPagedThreads, stream, a) != hipSuccess) return FUSED_MHA_ERR_LAUNCH;
  if (!p.shared) return FUSED_MHA_OK;
  const int rows = a.tokens * a.head;
  return launch(paged_join_kernel<D, BF>, dim3(p.join_grid(rows)), 256, stream, a, p.place_rows(), p.join_rows(rows)) == hipSuccess
             ? FUSED_MHA_OK : FUSED_MHA_ERR_LAUNCH;
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
  if ((tokens + 3) / 4 > kMostGroups) return FUSED_MHA_ERR_TOO_LARGE;
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
  if (rows >= (1L << 30) || blocks * b->batch > kMostGroups / 2) return FUSED_MHA_ERR_TOO_LARGE;
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
  if (head > (1 << 16) || all_tokens(b) >= (1L << 30) || all_tokens(b) * head >= (1L << 30)) return FUSED_MHA_ERR_TOO_LARGE;
  const Launch p = plan(c, b, head, max_new);
  // the line's length fits 62 bits: an item weighs up to four for each key and new token
  const double weight = 4. * ((double)b->table_width * c->page_size + 128 + b->tokens);
  if (p.items >= (1L << 30) || p.items * weight >= 0x1p61) return FUSED_MHA_ERR_TOO_LARGE;
  return p.grid() > kMostGroups || p.join_grid(all_tokens(b) * head) > kMostGroups ? FUSED_MHA_ERR_TOO_LARGE : FUSED_MHA_OK;
}

size_t paged_mha_forward_workspace_bytes(const paged_mha_cache* c, const paged_mha_batch* b, int head, int max_new) {
  return check_forward(c, b, head, max_new) ? 0 : workspace_bytes_of(plan(c, b, head, max_new), c->d, all_tokens(b) * head);
}

int paged_mha_forward(const paged_mha_cache* c, const paged_mha_batch* b, const void* q, const fused_mha_strides* q_st, void* o,
                      int head, int max_new, float scale, int causal, int zero_rest, void* workspace, size_t workspace_bytes,
                      void* stream) {
  if (const int rc = check_forward(c, b, head, max_new)) return rc;
  if (!q || !q_st || !o) return FUSED_MHA_ERR_NULL_POINTER;
  if (!isfinite(scale)) return FUSED_MHA_ERR_BAD_SCALE;
  if (bad_strides(q_st)) return FUSED_MHA_ERR_BAD_STRIDE;
  const Launch p = plan(c, b, head, max_new);
  const size_t wanted = workspace_bytes_of(p, c->d, all_tokens(b) * head);
  if (wanted && !workspace) return FUSED_MHA_ERR_NULL_POINTER;
  if (workspace_bytes < wanted) return PAGED_MHA_ERR_WORKSPACE;
  if (misaligned(q) || misaligned(o) || misaligned(workspace)) return FUSED_MHA_ERR_MISALIGNED;
  const int bytes = c->cache_type == PAGED_MHA_E4M3 ? 1 : 2;
  PagedArgs a{};
  a.q = (const char*)q, a.k = (const char*)c->key, a.v = (const char*)c->value, a.o = (char*)o;
  a.k_scale = (const unsigned char*)c->key_scale, a.v_scale = (const unsigned char*)c->value_scale;
  a.table = b->page_table, a.keys = b->cache_seqlens, a.ends = b->cu_seqlens ? b->cu_seqlens + 1 : nullptr;
  a.part_o = (float*)workspace;
  a.part_ml = (float2*)((char*)workspace + (size_t)2 * kPagedGroups * p.place_rows() * c->d * 4);
  a.places = (int2*)(a.part_ml + (size_t)2 * kPagedGroups * p.place_rows());
  a.ks = in_bytes(c->key_strides, bytes), a.vs = in_bytes(c->value_strides, bytes);
  a.kss = in_bytes(c->key_scale_strides, 1), a.vss = in_bytes(c->value_scale_strides, 1);
  a.q_batch = a.ends ? 0 : q_st->batch * 2, a.q_seq = q_st->seq * 2, a.q_head = q_st->head * 2;
  a.table_stride = b->table_stride;
  a.batch = b->batch, a.new_tokens = b->tokens, a.tokens = (int)all_tokens(b);
  a.head = head, a.kv_head = FmhaDivisor(c->kv_head), a.pages = c->pages, a.width = b->table_width;
  a.group = FmhaDivisor(head / c->kv_head), a.page_size = FmhaDivisor(c->page_size);
  a.c = scale * kLog2e;
  a.causal = causal != 0, a.zero_rest = zero_rest != 0 && a.ends;
  a.shared = p.shared;
  a.step[0] = paged_step(p.few, head / c->kv_head, p.many && p.few && bytes == 1 ? 2 : 4), a.step[1] = paged_step(kManyRows, head / c->kv_head, 4);
  if (p.many) fits(c, c->key_strides, bytes, a.k_shift), fits(c, c->value_strides, bytes, a.v_shift);
  return with_types(c, [&](auto d, auto bf, auto q8) {
    constexpr int D = decltype(d)::value;
    constexpr bool BF = decltype(bf)::value != 0, Q8 = decltype(q8)::value != 0;
    const hipStream_t st = (hipStream_t)stream;
    if (p.many) return p.few ? launch_forward<D, kFewRows, true, BF, Q8>(p, a, st) : launch_forward<D, 0, true, BF, Q8>(p, a, st);
    return p.few == 16 ? launch_forward<D, 16, false, BF, Q8>(p, a, st) : launch_forward<D, kFewRows, false, BF, Q8>(p, a, st);
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
    case FUSED_MHA_ERR_BAD_STRIDE: return "strides must be non-negative and not too large, with rows on 16-byte boundaries";
    case PAGED_MHA_ERR_BAD_TYPE: return "types must be fp16 or bf16, the cache of the same type or e4m3 with scales";
    case PAGED_MHA_ERR_BAD_PAGE_SIZE: return "page size must be a multiple of 16";
    case PAGED_MHA_ERR_BAD_GROUP: return "query heads must be a multiple of key heads";
    case PAGED_MHA_ERR_WORKSPACE: return "the workspace is too small";
    default: return "unknown error";
  }
}

}  // extern "C"
