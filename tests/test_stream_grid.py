"""How many blocks or clusters go through streamed rows, checked on the host function: no GPU needed."""
from __future__ import annotations

import subprocess

import pytest

from conftest import spmd_mod

PROGRAM = r"""
#include <cstdio>
#include "layer_norm.cuh"
int main() {
  for (int most = 0; most <= 40; ++most)
    for (int w = 1; w <= 8; w *= 2)
      for (int groups = 1; groups <= 256; groups *= 2)
        for (int64_t rows = 1; rows < 100000; rows = rows * 3 + 1)
          std::printf("%d %d %d %lld %d\n", most, w, groups, (long long)rows, spmdb200::stream_grid(rows, groups, most, w));
}
"""


def test_stream_grid_is_never_empty(tmp_path):
    """At least one block, also where fewer than a vector's elements are resident at once (a part of a GPU); a block
    either has one round of rows, or a stride of rows that is a multiple of w."""
    b = spmd_mod("build")
    try:
        nvcc = b.nvcc()
    except RuntimeError:
        pytest.skip("no nvcc")
    src, exe = tmp_path / "grid.cu", tmp_path / "grid"
    src.write_text(PROGRAM)
    r = subprocess.run([nvcc, *b.ARCH, "-O1", "-std=c++17", "--expt-relaxed-constexpr", f"-I{b.INCLUDE}", f"-I{b.CSRC}", str(src),
                        "-o", str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    lines = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60).stdout.splitlines()
    assert len(lines) > 10000
    for line in lines:
        most, w, groups, rows, grid = map(int, line.split())
        assert 1 <= grid <= max(most, w), line
        assert grid * groups >= rows or grid * groups % w == 0, line
        assert (grid - 1) * groups < rows, line  # every block has a row: partial rows are counted by it
