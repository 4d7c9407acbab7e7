// How the rows and keys of a batch over a paged cache are shared out among work groups: arithmetic for the host and the device.
#ifndef PAGED_PLAN_H_
#define PAGED_PLAN_H_

#include "block_map.h"

// Rows of a sequence and key head: its new tokens times the query heads of the key head, token by token.  A block is a number
// of neighbouring rows, an item a block of one sequence and key head, a part some of the key tiles of an item: the unit of
// work of a work group.  All items of a sequence have the same number of parts, numbered key head by key head, block by block.
constexpr int kPagedTile = 64;  // keys

FMHA_HOST_DEVICE int paged_tiles(int keys) { return (keys + kPagedTile - 1) / kPagedTile; }

FMHA_HOST_DEVICE int paged_blocks(int rows, int rows_of_block) { return (rows + rows_of_block - 1) / rows_of_block; }

// Tiles of a part, of so many in all that there are about `target` parts, but none of fewer than `least` tiles.
FMHA_HOST_DEVICE int paged_tiles_of_part(long tiles, int target, int least) {
  const long even = (tiles + target - 1) / target;
  return even > least ? (int)even : least;
}

// Parts of an item of so many tiles: at least one, which writes the result of items without keys.
FMHA_HOST_DEVICE int paged_parts(int tiles, int tiles_of_part) { return tiles <= tiles_of_part ? 1 : (tiles + tiles_of_part - 1) / tiles_of_part; }

// Tiles first .. end-1 of part p; none where there are fewer tiles than parts.
FMHA_HOST_DEVICE void paged_part(int tiles, int parts, int p, int& first, int& end) {
  const int each = tiles / parts, more = tiles - each * parts;
  first = p * each + (p < more ? p : more);
  end = first + each + (p < more ? 1 : 0);
}

// Keys that the last of new tokens 0 .. i sees.
FMHA_HOST_DEVICE int paged_visible(int keys, int new_tokens, int i, bool causal) {
  const int seen = causal ? keys - new_tokens + i + 1 : keys;
  return seen < 0 ? 0 : seen;
}

// Work group w of a launch takes part paged_spread(w, parts), if that is one: neighbouring parts, which read the same keys, go to the
// same XCD (work groups go round-robin over the 8).  The launch has at least 8 * ceil(parts / 8) work groups.
FMHA_HOST_DEVICE int paged_spread(int w, int parts) {
  const int run = (parts + 7) >> 3;
  return (w >> 3) < run ? (w & 7) * run + (w >> 3) : parts;
}

#endif  // PAGED_PLAN_H_
