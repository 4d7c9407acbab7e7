// How the rows and keys of a batch over a paged cache are shared out among work groups: arithmetic for the host and the device.
#ifndef PAGED_PLAN_H_
#define PAGED_PLAN_H_

#include "block_map.h"

// Rows of a sequence and key head: its new tokens times the query heads of the key head, token by token.  A block is a number
// of neighbouring rows, an item a block of one sequence and key head with the tiles of keys that it sees.  kPagedGroups work groups
// share the items in one of three ways, whichever takes the longest of them the least time; none needs to know what others do:
//
//   stretches  Items stand in a line, sequence by sequence, key head by key head, block by block, each as long as its work (its
//              weight), and each work group gets a stretch of the line of the same length: the end of an item that begins in an
//              earlier stretch, whole items, and the beginning of one that goes on in the next.  An item that lies in several
//              stretches is joined afterwards, part by part.
//   parts      The same with items rounded up to whole stretches, so that none begins inside of one.
//   whole      Items in rounds, the ones that see most first, key heads next to each other; nothing to join.
constexpr int kPagedTile = 64;  // keys

FMHA_HOST_DEVICE int paged_tiles(int keys) { return (keys + kPagedTile - 1) / kPagedTile; }

FMHA_HOST_DEVICE int paged_blocks(int rows, int rows_of_block) { return (rows + rows_of_block - 1) / rows_of_block; }

// Keys that the last of new tokens 0 .. i sees.
FMHA_HOST_DEVICE int paged_visible(int keys, int new_tokens, int i, bool causal) {
  const int seen = causal ? keys - new_tokens + i + 1 : keys;
  return seen < 0 ? 0 : seen;
}

// Weights of the items of a sequence and key head: of block k `first + step * (k + 1)`.
struct PagedLine {
  long first;
  int step, blocks;
  FMHA_HOST_DEVICE long before(int k) const { return k * first + (long)step * k * (k + 1) / 2; }
  FMHA_HOST_DEVICE long of(int k) const { return first + (long)step * (k + 1); }
  FMHA_HOST_DEVICE long all() const { return before(blocks); }
};
// About the keys that a block sees, and something for its beginning and end, times the weight of a key.  step: 0 without a causal
// mask, else paged_step, which divides.
FMHA_HOST_DEVICE int paged_step(int rows_of_block, int group, int of_key) { return of_key * rows_of_block / group; }
template <typename Int>  // int or FmhaDivisor
FMHA_HOST_DEVICE PagedLine paged_line(int keys, int new_tokens, const Int& group, int step, int rows_of_block, int overhead, int of_key) {
  const int hidden = step == 0 ? 0 : new_tokens < keys ? new_tokens : keys;
  return PagedLine{of_key * (long)(keys - hidden + overhead), step, paged_blocks(new_tokens * group, rows_of_block)};
}
// Parts of an item of that weight, none of them longer than 1 / per_length.
FMHA_HOST_DEVICE int paged_parts(float weight, float per_length) { return (int)(weight * per_length) + 1; }

// n / d where that is below 2^20: by floats, put right.
template <typename Int>  // int or long
FMHA_HOST_DEVICE int paged_divide(Int n, Int d) {
  int q = (int)((float)n / (float)d);
  if (q * d > n) --q;
  if ((q + 1) * d <= n) ++q;
  return q;
}

// Tiles of block `block` of a sequence's rows: those that the last of its rows sees.
template <typename Int>
FMHA_HOST_DEVICE int paged_tiles_of(int keys, int new_tokens, const Int& group, int rows_of_block, int block, bool causal) {
  const int rows = new_tokens * group, end = (block + 1) * rows_of_block, last = (rows < end ? rows : end) - 1;
  return paged_tiles(paged_visible(keys, new_tokens, last / group, causal));
}

// Length of a stretch: the same for up to kPagedGroups of them, which is as many work groups as the device runs at a time, but
// not so short that a work group has little else to do than to begin and end.  With 128, 256 and 512 keys at least, us: one token over
// 1500 keys 10.7, 11.5, 12.0; 64 over 200, 8 key heads, which 128 splits, 16.0, 12.2, 11.6; 200 of those 32.4, 26.9, 26.9.
constexpr int kPagedGroupsLog = 9, kPagedGroups = 1 << kPagedGroupsLog;
constexpr int kPagedLeastLog = 10, kPagedLeast = 1 << kPagedLeastLog;  // 256 keys
FMHA_HOST_DEVICE long paged_stretch(long all) {
  const long even = (all + kPagedGroups - 1) >> kPagedGroupsLog;
  return even > kPagedLeast ? even : kPagedLeast;
}
// How many there are, or a few more.
FMHA_HOST_DEVICE int paged_stretches(long all, long length) {
  return length > kPagedLeast ? kPagedGroups : (int)((all + kPagedLeast - 1) >> kPagedLeastLog);
}

// Block in which position x (from 0 to all() - 1) of a key head's line lies.
FMHA_HOST_DEVICE int paged_block_at(const PagedLine& line, long x) {
  int lo = 0, hi = line.blocks - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (line.before(mid) <= x) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// The tile at which a stretch that begins or ends `into` an item of that weight begins or ends.
FMHA_HOST_DEVICE int paged_tile_at(int tiles, long into, long weight) {
  if (into <= 0) return 0;
  if (into >= weight) return tiles;
  const int at = (int)((float)into * ((float)tiles / (float)weight));  // grows with `into`, the same on both sides
  return at < tiles ? at : tiles;
}

// Where parts of an item that begins in stretch r lie: stretch s has two places, 2 s for the end of an item and 2 s + 1 for the
// beginning of one.  An item that is all of a stretch and more, begun before, is an end.
FMHA_HOST_DEVICE int paged_place(int r, int part) { return 2 * (r + part) + (part == 0 ? 1 : 0); }

// In the functions below `same` returns its argument, which all lanes of a wave have: the kernels put it into a scalar register.

// What a stretch from x to `end` takes of the item at x: its block and key head, tiles t0 .. t1 - 1, whether it begins here and is whole,
// how many parts it has if it begins here, and the place of this one.  `begin`: where the sequence's first key head lies in the line.
struct PagedShare {
  int head, block, t0, t1, parts, place;
  bool opens, whole;
  long item, weight;
};
template <typename Same>
FMHA_HOST_DEVICE void paged_item_at(const PagedLine& line, long begin, long x, PagedShare& r, Same same) {
  const long of_head = line.all();
  r.head = same(paged_divide(x - begin, of_head));
  const long from = begin + r.head * of_head;
  r.block = line.blocks == 1 ? 0 : same(paged_block_at(line, x - from));
  r.item = from + line.before(r.block), r.weight = line.of(r.block);
}
template <typename Same>
FMHA_HOST_DEVICE void paged_share_of_stretch(int tiles, long x, long end, long length, int stretch, PagedShare& r, Same same) {
  r.t0 = same(paged_tile_at(tiles, x - r.item, r.weight));
  r.t1 = same(paged_tile_at(tiles, end - r.item, r.weight));
  r.opens = same((int)(r.item >= x));
  r.whole = r.opens && same((int)(r.item + r.weight <= end));
  r.parts = r.whole || !r.opens ? 1 : same(paged_divide(r.item + r.weight - 1, length)) - stretch + 1;
  r.place = paged_place(stretch, r.opens ? 0 : 1) - (r.opens ? 0 : 2);
}

// Part `at` of a sequence's, where each of its items has `each`.
template <typename Same>
FMHA_HOST_DEVICE void paged_part_item(int at, int blocks, int each, int& block, int& head, int& part, Same same) {
  const int of_head = blocks * each;
  head = same(paged_divide(at, of_head));
  block = same(paged_divide(at - head * of_head, each));
  part = at - head * of_head - block * each;
}
// First tile of a part, or the end of the last one; per: about tiles / parts, the same for all of them.
FMHA_HOST_DEVICE int paged_part_tile(int tiles, int part, int parts, float per) {
  return part == 0 ? 0 : part == parts ? tiles : (int)((float)part * per);
}

// Item that work group w takes in a round of whole ones: as the persistent kernels for equal lengths, or, if there is one round only,
// as those of which two share a CU.
FMHA_HOST_DEVICE int paged_whole(int round, int w, int items) {
  return items <= kPagedGroups ? round == 0 && w < items ? fmha_paired_block(w, items) : items : fmha_persistent_block(round, w, kPagedGroups);
}
// Item `at` of a sequence's: its block, the last one first, and key head.
template <typename Int>
FMHA_HOST_DEVICE void paged_whole_item(int at, int blocks, const Int& kv_heads, int& block, int& head) {
  const int level = at / kv_heads;
  block = blocks - 1 - level;
  head = at - level * (int)kv_heads;
}

// Work group w of a launch has stretch paged_spread(w, stretches), if that is one: neighbouring stretches, which read the same keys,
// go to the same XCD (work groups go round-robin over the 8).  The launch has at least 8 * ceil(stretches / 8) work groups.
FMHA_HOST_DEVICE int paged_spread(int w, int stretches) {
  const int run = (stretches + 7) >> 3;
  return (w >> 3) < run ? (w & 7) * run + (w >> 3) : stretches;
}

// What the table of a row's parts says of an item that begins in stretch r: the row of its place, with slot_rows rows to a place, less
// slot_rows.  Whole items, of which there may be many more than stretches, have no place.
FMHA_HOST_DEVICE int paged_first_row(int r, int parts, int slot_rows) { return parts > 1 ? 2 * r * slot_rows : 0; }
// Whether a row's parts lie among the places, of slot_rows rows each: the first at row `at` + slot_rows, the next ones twice that apart.
FMHA_HOST_DEVICE bool paged_parts_fit(int at, int parts, int slot_rows) {
  return at >= 0 && parts > 1 && at + 2l * (parts - 1) * slot_rows < 2l * kPagedGroups * slot_rows;
}

#endif  // PAGED_PLAN_H_
