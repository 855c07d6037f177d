"""The deal of sparse attention's key tiles to workgroups (csrc/tile_runs.h, which the plan
and the kernel share), on the CPU: the kernel's walk over units and runs in plain C++."""
import ctypes
import os
import random
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gllm_amd", "csrc")

# Walks every run as sparse_tile_kernel does.  Returns 0, or what does not hold.
WALK = r"""
#include <algorithm>
#include <cstdio>
#include <vector>
#include "tile_runs.h"
using namespace gllm;

extern "C" int walk(int64_t round, int32_t bs, int32_t units, const int32_t* tiles, int64_t all, int64_t* most) {
  int64_t C = 0;
  for (int u = 0; u < units; ++u) C += tiles[u];
  if (all < C) return 1;
  const int64_t W = tile_runs(all, round, bs), runs = std::min(W, tile_runs(C, round, bs));
  if (runs < 1 || runs > C || runs != tile_runs(C, round, bs)) return 2;
  std::vector<char> used((size_t)run_slots(W, units), 0);
  std::vector<std::vector<int64_t>> slots(units);
  std::vector<int64_t> seen(units, 0);
  for (int64_t b = 0; b < runs; ++b) {
    const int64_t lo = run_start(C, runs, b), hi = run_start(C, runs, b + 1);
    if (lo >= hi || run_of(C, runs, lo) != b || run_of(C, runs, hi - 1) != b) return 3;
    int u = 0;
    int64_t s0 = 0;
    while (s0 + tiles[u] <= lo) s0 += tiles[u++];
    int64_t slot = part_slot(runs, units, b, u, true);
    for (int64_t s = lo; s < hi; ++u) {
      const int64_t c = tiles[u], end = std::min(hi, s0 + c);
      const bool whole = s == s0 && end == s0 + c;
      // the blocks whose ids the workgroup holds
      const int64_t first = 64 * (s - s0) / bs, last = (64 * (end - s0) - 1) / bs;
      *most = std::max(*most, last - first + 1);
      if (last - first + 1 > kRunCache) return 4;
      if (s - s0 != seen[u]) return 5;
      seen[u] = end - s0;
      if (!whole) {
        if (slot < 0 || slot >= (int64_t)used.size()) return 6;
        if (used[slot]) return 7;
        used[slot] = 1;
        slots[u].push_back(slot);
      }
      s0 += c;
      s = end;
      slot = units < runs ? slot + 1 : slot | 1;
    }
  }
  int64_t s0 = 0;
  for (int u = 0; u < units; s0 += tiles[u++]) {
    if (seen[u] != tiles[u]) return 8;
    const TileParts p = unit_parts(C, runs, units, u, s0, tiles[u]);
    if (p.count != std::max<int64_t>(1, (int64_t)slots[u].size()) || slots[u].size() == 1) return 9;
    for (size_t k = 0; k < slots[u].size(); ++k)
      if (slots[u][k] != (k == 0 ? p.first : p.rest + ((int64_t)k - 1) * p.step)) return 10;
  }
  return 0;
}
extern "C" int64_t group_run(int64_t group, int64_t runs) { return run_of_group(group, runs); }
extern "C" int64_t most_tiles(int32_t bs) { return most_run_tiles(bs); }
extern "C" int64_t runs_of(int64_t C, int64_t round, int32_t bs) { return tile_runs(C, round, bs); }
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("runs")
    (d / "walk.cpp").write_text(WALK)
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", "-shared", "-fPIC", f"-I{CSRC}", str(d / "walk.cpp"), "-o",
                    str(d / "walk.so")], check=True)
    so = ctypes.CDLL(str(d / "walk.so"))
    so.most_tiles.restype = so.runs_of.restype = ctypes.c_int64
    so.group_run.restype, so.group_run.argtypes = ctypes.c_int64, [ctypes.c_int64, ctypes.c_int64]
    so.runs_of.argtypes = [ctypes.c_int64, ctypes.c_int64, ctypes.c_int32]
    so.walk.argtypes = [ctypes.c_int64, ctypes.c_int32, ctypes.c_int32, ctypes.c_void_p, ctypes.c_int64, ctypes.c_void_p]
    return so


def _walk(lib, round_, bs, tiles, more=0):
    arr, most = (ctypes.c_int32 * len(tiles))(*tiles), ctypes.c_int64(0)
    rc = lib.walk(round_, bs, len(tiles), arr, sum(tiles) + more, ctypes.byref(most))
    assert rc == 0, f"check {rc}: round {round_}, blocks of {bs}, {len(tiles)} units of {tiles[:20]}, {more} more planned"
    return most.value


@pytest.mark.parametrize("bs", [16, 48, 64, 80, 112, 1040, 65536])
def test_every_small_deal(lib, bs):
    rng = random.Random(bs)
    for round_ in (1, 2, 3, 7, 8):
        for units in (1, 2, 3, 5, 9, 17, 40):
            for top in (1, 3, 9, 300, 3000):
                for _ in range(3):
                    tiles = [rng.randint(1, top) for _ in range(units)]
                    _walk(lib, round_, bs, tiles, rng.choice([0, 0, 1, 7, sum(tiles), 20 * sum(tiles)]))


@pytest.mark.parametrize("bs", [16, 48, 64, 80, 112])
@pytest.mark.parametrize("round_", [1, 8, 256, 304])
def test_full_runs_and_rounds(lib, bs, round_):
    """Runs as long as they get, one tile either side of a round's end, in one unit and in
    several: their blocks fit what a workgroup holds."""
    full, longest = round_ * lib.most_tiles(bs), 0
    for C in (full - 1, full, full + 1, 2 * full, 2 * full + 1, 5 * full + 3):
        assert lib.runs_of(C, round_, bs) == min(max(1, C // 4), -(-C // full) * round_)
        longest = max(longest, _walk(lib, round_, bs, [C]))
        longest = max(longest, _walk(lib, round_, bs, [1, C - 2, 1]) if C > 2 else 0)
        third = C // 3
        longest = max(longest, _walk(lib, round_, bs, [third + 1, third, C - 2 * third - 1]))
    assert 1015 < longest <= 1024


def test_more_units_than_runs(lib):
    rng = random.Random(0)
    for units in (255, 256, 257, 1000, 4000):
        for top in (1, 4, 60):
            tiles = [rng.randint(1, top) for _ in range(units)]
            _walk(lib, 256, 16, tiles, rng.choice([0, 3 * sum(tiles)]))


def test_runs_grow_with_the_tiles(lib):
    """The kernel counts the tiles that there are; the plan's workgroups, from the most that
    there can be, are as many or more."""
    for bs in (16, 112):
        for round_ in (3, 256):
            last = 0
            for C in sorted({1, 2, 5, 1023, 1024, 1025, *range(1, 40 * lib.most_tiles(bs) * round_, 977)}):
                n = lib.runs_of(C, round_, bs)
                assert n >= last
                last = n


@pytest.mark.parametrize("runs", [1, 7, 8, 9, 250, 256, 1024, 1280])
@pytest.mark.parametrize("planned", [1, 2, 5])
def test_every_xcd_has_its_share_of_runs(lib, runs, planned):
    """Workgroups go to the 8 XCDs in turn.  A plan counts the most runs that there can be; the
    ones that there are must not leave XCDs idle."""
    groups = [lib.group_run(g, runs) for g in range(runs * planned)]
    assert sorted(r for r in groups if r < runs) == list(range(runs))
    share = [sum(r < runs for r in groups[x::8]) for x in range(8)]
    assert max(share) - min(share) <= 1
    if runs % 8 == 0:                                   # neighbours together
        for x in range(8):
            assert sorted(r for r in groups[x::8] if r < runs) == list(range(x * runs // 8, (x + 1) * runs // 8))
