"""Items of the launches for few tokens over the blocks (CPU): the kernel's own arithmetic (csrc/few_split.cuh), compiled for the
host and walked the way the blocks walk it."""

import ctypes
import random
import subprocess
from pathlib import Path

import numpy as np
import pytest

CSRC = Path(__file__).resolve().parents[1] / "dist_moe_b200" / "csrc"

HARNESS = r"""
#include "few_split.cuh"
extern "C" void walk(int64_t strips, int length, int grid, int64_t* begin, int64_t* end, int* first_block, int* last_block, int64_t* place) {
  const dm::FewSplit s(strips, length, grid);
  for (int b = 0; b < grid; ++b) begin[b] = s.begin(b), end[b] = s.end(b);
  for (int64_t q = 0; q < strips; ++q) {
    first_block[q] = s.first_block(q), last_block[q] = s.last_block(q);
    for (int b = first_block[q]; b <= last_block[q]; ++b) place[q * grid + b] = s.place(b, q);
  }
}
"""


@pytest.fixture(scope="module")
def walk(tmp_path_factory):
    folder = tmp_path_factory.mktemp("few_split")
    (folder / "harness.cpp").write_text(HARNESS)
    subprocess.run(["g++", "-std=c++17", "-O2", "-shared", "-fPIC", "-x", "c++", str(folder / "harness.cpp"), f"-I{CSRC}",
                    "-o", str(folder / "harness.so")], check=True)
    lib = ctypes.CDLL(str(folder / "harness.so"))

    def call(strips, length, grid):
        out = [np.full(grid, -1, np.int64), np.full(grid, -1, np.int64), np.full(strips, -1, np.int32), np.full(strips, -1, np.int32),
               np.full(strips * grid, -1, np.int64)]
        lib.walk(ctypes.c_int64(strips), length, grid, *(a.ctypes.data_as(ctypes.c_void_p) for a in out))
        return out

    return call


# fewer items than blocks, one item, whole strips alone, strips over many blocks; then sizes at random
SHAPES = [(1, 1, 148), (1, 3, 148), (2, 1, 148), (147, 1, 148), (149, 1, 148), (64, 66, 148), (1, 500, 148), (300, 8, 1), (5, 7, 2)]
_rng = random.Random(4)
SHAPES += [(_rng.randint(1, 120), _rng.randint(1, 60), _rng.choice([148, 132, 7])) for _ in range(60)]


@pytest.mark.parametrize("strips,length,grid", SHAPES)
def test_every_item_once_and_parts_meet(walk, strips, length, grid):
    begin, end, first, last, place = walk(strips, length, grid)
    items = strips * length
    assert begin[0] == 0 and end[-1] == items and (begin[1:] == end[:-1]).all() and (end >= begin).all()
    assert (end - begin).max() - (end - begin)[end > begin].min() <= 1  # even
    parts = {}
    for b in range(grid):
        for q in {int(i) // length for i in range(begin[b], end[b])}:
            parts.setdefault(q, []).append(b)
    taken = {}
    for q in range(strips):
        assert parts[q] == list(range(first[q], last[q] + 1))  # as many arrivals as the last one waits for
        if len(parts[q]) > 1:
            for b in parts[q]:
                at = int(place[q * grid + b])
                assert 0 <= at < 2 * grid and taken.setdefault(at, q) == q
                assert at // 2 == b
    assert len(taken) == sum(len(b) for b in parts.values() if len(b) > 1)
