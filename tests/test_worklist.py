"""The attention kernels' work-list arithmetic, compiled for the host with
overflow checks: lengths and row starts from device memory may hold anything."""

from __future__ import annotations

import itertools
import pathlib
import subprocess

import pytest

CSRC = pathlib.Path(__file__).resolve().parent.parent / "se12_b200" / "csrc"
MAX = 2**31 - 1

PROGRAM = r"""
#include <cstdio>
#include "se12_worklist.h"
using namespace se12;
int main() {
  int start, stop, len, tokens, capacity, group, window, chunk, rows, tile, heads, cost;
  while (std::scanf("%d %d %d %d %d %d %d %d %d %d %d %d", &start, &stop, &len, &tokens, &capacity, &group, &window, &chunk, &rows,
                    &tile, &heads, &cost) == 12) {
    const ListSizes z{tokens, capacity, group, window};
    const SeqRows s = sequence_rows(start, stop, len, z);
    const SeqWork w = sequence_work(s, z, chunk, rows);
    const int limit = static_cast<int>(kWorkLimit / heads);
    const int one = times_work(w.chunks + cost, w.tiles, limit), two = add_work(one, one, limit);
    std::printf("%d %d %d %d %d %d %d %d %d", first_row(start, z), s.tokens, s.first, s.length, w.low, w.chunks, w.tiles, one, two);
    if (w.tiles) {
      const TileSpan p = tile_span(s, tile % w.tiles, rows, z, chunk);
      std::printf(" %d %d %d %d %d", p.low, span_end(s, p.pos_max), p.chunks, p.pos_min, p.pos_max);
    }
    std::printf("\n");
  }
}
"""

STARTS = [(0, 1), (0, 5), (3, 3), (-7, 4), (4, -7), (2, MAX), (-MAX - 1, MAX), (100, 90), (1000, 5000)]
LENS = [0, 1, 15, 16, 17, 700, 1 << 30, MAX, -1, -MAX - 1]
BATCHES = [(5, 16, 1, 0), (5, 16, 8, 3), (1000, 4096, 11, 4095), (1000, 4096, 128, 1), (1 << 20, MAX - 4096, 8, 0),
           (1 << 20, MAX - 4096, 8, MAX - 4097), (1 << 30, 1 << 30, 1, 77)]
TILES = [(16, 8, 0), (32, 16, 1), (64, 128, 3), (128, 128, 10**6)]


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    directory = tmp_path_factory.mktemp("worklist")
    (directory / "list.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover=all", f"-I{CSRC}",
                    "-o", str(directory / "list"), str(directory / "list.cpp")], check=True, capture_output=True)
    return directory / "list"


def clamp(x, low, high):
    return max(low, min(x, high))


def test_counts_at_the_bounds(program):
    cases = [(start, stop, length, *batch, *tile, heads, cost) for (start, stop), length, batch, tile, (heads, cost)
             in itertools.product(STARTS, LENS, BATCHES, TILES, [(1, 8), (8, 3), (1000, 8)])]
    cases = [c for c in cases if c[3] * c[5] <= 1 << 30]  # as the host sees to
    run = subprocess.run([str(program)], input="\n".join(" ".join(map(str, c)) for c in cases), capture_output=True, text=True)
    assert run.returncode == 0, run.stderr
    lines = run.stdout.splitlines()
    assert len(lines) == len(cases)
    for case, line in zip(cases, lines):
        start, stop, length, tokens, capacity, group, window, chunk, rows, tile, heads, cost = case
        got = list(map(int, line.split()))
        begin = clamp(start, 0, tokens)
        count = clamp(stop, begin, tokens) - begin
        held = max(length, 0)
        first, held = held - count, min(held, capacity)
        assert got[:4] == [begin, count, first, held], case
        visible = max(first - window + 1, 0) if window else 0
        low, chunks, tiles, one, two = got[4:9]
        assert low % chunk == 0 and low <= min(visible, held) < low + chunk
        assert chunks == max(-(-(held - low) // chunk), 1) and tiles == -(-count * group // rows)
        limit = ((1 << 31) - (1 << 20)) // heads
        assert one == min((chunks + cost) * tiles, limit) and two == min(2 * one, limit)
        assert 0 <= two * heads <= MAX
        if not tiles:
            continue
        tile %= tiles
        low, end, chunks, pos_min, pos_max = got[9:]
        assert pos_min == first + tile * rows // group and pos_max == first + min(tile * rows + rows - 1, count * group - 1) // group
        assert end == min(pos_max + 1, held)
        visible = max(pos_min - window + 1, 0) if window else 0
        assert low % chunk == 0 and low <= min(visible, held) < low + chunk
        assert chunks == max(-(-(end - low) // chunk), 1)
