"""CPU tests of csrc/paged_plan.h, the arithmetic by which work groups find their share of a batch: the functions that the kernels
call, in programs of their own."""
import os
import subprocess

import abi

CSRC = os.path.join(abi.ROOT, "flash-attention-v100_amd", "csrc")


def run(tmp_path, body):
    """What a program prints; it ends early where signed numbers overflow."""
    src, exe = tmp_path / "plan.cpp", tmp_path / "plan"
    src.write_text('#include <cmath>\n#include <cstdio>\n#include <vector>\n#include "paged_plan.h"\n' + body)
    subprocess.check_call(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-ftrapv", "-I", CSRC, str(src), "-o", str(exe)])
    return subprocess.run([str(exe)], stdout=subprocess.PIPE).stdout.decode()


def test_rows_of_places(tmp_path):
    """Where the table says that parts begin; items that have none are up to 2^30."""
    out = run(tmp_path, r"""
int main() {
  for (int rows : {16, 32, 128}) {
    for (int first = 0; first < kPagedGroups; ++first)
      if (paged_first_row(first, 2, rows) + rows != paged_place(first, 0) * rows) return puts("place"), 1;
    for (int item : {1 << 23, 1 << 24, (1 << 30) - 1})
      if (paged_first_row(item, 1, rows) != 0) return puts("whole"), 1;
  }
  puts("ok");
}
""")
    assert out == "ok\n"


BATCHES = r"""
struct Seq { int n, keys; };
struct Batch {
  int kv, group, rows_of_block;
  bool causal;
  std::vector<Seq> seqs;
  int tiles(const Seq& s, int block) const { return paged_tiles_of(s.keys, s.n, group, rows_of_block, block, causal); }
  int blocks(const Seq& s) const { return paged_blocks(s.n * group, rows_of_block); }
  PagedLine line(const Seq& s) const { return paged_line(s.keys, s.n, group, causal ? paged_step(rows_of_block, group, 4) : 0, rows_of_block, 64, 4); }
};
unsigned seed = 1;
int rnd(int n) { seed = seed * 1664525u + 1013904223u; return (int)((seed >> 8) % (unsigned)n); }
Batch random_batch() {
  Batch b{1 + rnd(4), 1 + rnd(9), rnd(3) == 0 ? 16 : rnd(2) ? 32 : 128, rnd(2) != 0, std::vector<Seq>(1 + rnd(12))};
  for (Seq& s : b.seqs) s = {rnd(3) ? rnd(3) : rnd(300), rnd(3) ? rnd(500) : rnd(20000)};
  return b;
}
auto same = [](int x) { return x; };
// What has been taken of an item, one part after the other.
struct Taken { int upto = 0, parts = 0, first_row = 0; };
struct Items {
  const Batch& b;
  std::vector<std::vector<Taken>> of;
  std::vector<int> places = std::vector<int>(2 * kPagedGroups);
  explicit Items(const Batch& b) : b(b) {
    for (const Seq& s : b.seqs) of.emplace_back(b.kv * b.blocks(s));
  }
  Taken& at(int seq, int head, int block) { return of[seq][head * b.blocks(b.seqs[seq]) + block]; }
  // false: not the next part of the item, or not where the join looks for it
  bool take(int seq, const PagedShare& r, int stretch) {
    if (r.head < 0 || r.head >= b.kv || r.block < 0 || r.block >= b.blocks(b.seqs[seq])) return false;
    Taken& t = at(seq, r.head, r.block);
    if (r.opens != (t.parts == 0) || r.t0 != t.upto || r.t1 < r.t0) return false;
    if (r.opens) t.first_row = paged_first_row(stretch, r.parts, b.rows_of_block);
    if (r.opens && r.parts > 1 && !paged_parts_fit(t.first_row, r.parts, b.rows_of_block)) return false;
    if (!r.whole) {
      if (r.place < 0 || r.place >= 2 * kPagedGroups || places[r.place]++) return false;
      if (t.first_row + paged_place(0, t.parts) * b.rows_of_block != r.place * b.rows_of_block) return false;
    }
    t.upto = r.t1, ++t.parts;
    return true;
  }
  bool all_taken(int seq, int head, int block, int parts) { return at(seq, head, block).upto == b.tiles(b.seqs[seq], block) && at(seq, head, block).parts == parts; }
};
"""


def test_tiles_of_a_block(tmp_path):
    """As many as hold a key that one of its rows sees."""
    out = run(tmp_path, BATCHES + r"""
int main() {
  for (int i = 0; i < 4000; ++i) {
    Batch b = random_batch();
    const Seq s{1 + rnd(60), rnd(400)};
    for (int block = 0; block < b.blocks(s); ++block) {
      int last = -1;
      for (int row = block * b.rows_of_block; row < (block + 1) * b.rows_of_block && row < s.n * b.group; ++row)
        for (int key = 0; key < s.keys; ++key)
          if (!b.causal || key <= s.keys - s.n + row / b.group) last = key > last ? key : last;
      if (b.tiles(s, block) != last / kPagedTile + (last >= 0)) return puts("wrong"), 1;
    }
  }
  puts("ok");
}
""")
    assert out == "ok\n"


def test_stretches_take_every_tile_once(tmp_path):
    """In places of their own, where the join looks for them; a stretch has as large a share of an item's tiles as of its place in the
    line, but for the tile at each end."""
    out = run(tmp_path, BATCHES + r"""
int main() {
  for (int round = 0; round < 3000; ++round) {
    const Batch b = random_batch();
    Items items(b);
    std::vector<std::vector<int>> told;
    long all = 0;
    for (const Seq& s : b.seqs) {
      all += b.line(s).all() * b.kv;
      told.emplace_back(b.kv * b.blocks(s));
    }
    const long length = paged_stretch(all);
    const int stretches = paged_stretches(all, length);
    for (int s = 0; s < stretches; ++s) {
      const long end = (s + 1) * length < all ? (s + 1) * length : all;
      for (long x = s * length; x < end;) {
        long begin = 0;
        int seq = 0;
        for (; begin + b.line(b.seqs[seq]).all() * b.kv <= x; ++seq) begin += b.line(b.seqs[seq]).all() * b.kv;
        PagedShare r;
        paged_item_at(b.line(b.seqs[seq]), begin, x, r, same);
        if (r.weight <= 0 || r.item > x || r.item + r.weight <= x) return puts("item"), 1;
        const int tiles = b.tiles(b.seqs[seq], r.block);
        paged_share_of_stretch(tiles, x, end, length, s, r, same);
        if (!items.take(seq, r, s)) return puts("part"), 1;
        if (r.opens) told[seq][r.head * b.blocks(b.seqs[seq]) + r.block] = r.parts;
        const long from = x > r.item ? x : r.item, to = end < r.item + r.weight ? end : r.item + r.weight;
        if (std::fabs(r.t1 - r.t0 - (double)tiles * (to - from) / r.weight) > 1.01) return puts("share"), 1;
        x = r.item + r.weight;
      }
    }
    for (int seq = 0; seq < (int)b.seqs.size(); ++seq)
      for (int head = 0; head < b.kv; ++head)
        for (int block = 0; block < b.blocks(b.seqs[seq]); ++block)
          if (!items.all_taken(seq, head, block, told[seq][head * b.blocks(b.seqs[seq]) + block])) return puts("not whole"), 1;
  }
  puts("ok");
}
""")
    assert out == "ok\n"


def test_parts_take_every_tile_once(tmp_path):
    """Likewise, in equal parts but for a tile; the quotient of tiles and parts, which the device only has about, may be off by a few of its
    last bits."""
    out = run(tmp_path, BATCHES + r"""
int main() {
  for (int round = 0; round < 3000; ++round) {
    const Batch b = random_batch();
    Items items(b);
    // parts no longer than some length, the least for which there are places enough
    std::vector<int> each(b.seqs.size());
    int places;
    for (float length = 256 + rnd(2000);; length *= 1.25f) {
      places = 0;
      for (int i = 0; i < (int)each.size(); ++i) {
        const Seq s = b.seqs[i];
        each[i] = paged_parts(s.n ? 4.f * (s.keys + 64) : 0.f, 1.f / length);
        places += b.kv * b.blocks(s) * each[i];
      }
      if (places <= kPagedGroups || length > 1e6f) break;
    }
    if (places > kPagedGroups) continue;
    const float off = 1.f + (rnd(5) - 2) * 0x1p-23f;
    int at = 0;
    for (int i = 0; i < (int)each.size(); ++i) {
      const Seq s = b.seqs[i];
      const int count = b.kv * b.blocks(s) * each[i];
      for (int local = 0; local < count; ++local, ++at) {
        PagedShare r;
        int part;
        paged_part_item(local, b.blocks(s), each[i], r.block, r.head, part, same);
        const int tiles = b.tiles(s, r.block);
        const float per = (float)tiles * (1.f / each[i]) * off;
        r.t0 = paged_part_tile(tiles, part, each[i], per), r.t1 = paged_part_tile(tiles, part + 1, each[i], per);
        r.opens = part == 0, r.whole = each[i] == 1, r.parts = each[i], r.place = paged_place(at - part, part);
        if (!items.take(i, r, at)) return puts("part"), 1;
        if (std::fabs(r.t1 - r.t0 - (double)tiles / each[i]) > 1.01) return puts("share"), 1;
      }
    }
    for (int seq = 0; seq < (int)b.seqs.size(); ++seq)
      for (int head = 0; head < b.kv; ++head)
        for (int block = 0; block < b.blocks(b.seqs[seq]); ++block)
          if (!items.all_taken(seq, head, block, each[seq])) return puts("not whole"), 1;
  }
  puts("ok");
}
""")
    assert out == "ok\n"


def test_parts_of_the_longest_sequences(tmp_path):
    """Up to 2^24 tiles in up to 512 parts: every tile once."""
    out = run(tmp_path, r"""
int main() {
  for (int parts = 1; parts <= kPagedGroups; ++parts)
    for (int tiles : {0, 1, 2, parts - 1, parts, parts + 1, 1000, 65535, 65537, (1 << 24) - 1, 1 << 24})
      for (int bits = -2; bits <= 2; ++bits) {
        const float per = (float)tiles * (1.f / parts) * (1.f + bits * 0x1p-23f);
        for (int part = 0; part < parts; ++part)
          if (paged_part_tile(tiles, part + 1, parts, per) < paged_part_tile(tiles, part, parts, per)) return puts("back"), 1;
        if (paged_part_tile(tiles, 0, parts, per) != 0 || paged_part_tile(tiles, parts, parts, per) != tiles) return puts("ends"), 1;
      }
  puts("ok");
}
""")
    assert out == "ok\n"
