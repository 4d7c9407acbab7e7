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
