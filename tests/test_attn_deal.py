"""CPU tests of the walk over the few-row kernels' deal (csrc/kernels/attn_deal.h, compiled here), as the kernel takes it: the units are
summed from the counts first, and the counts read again along the walk."""
import ctypes
import subprocess

import numpy as np
import pytest

from saber_engine_amd import iu8

SOURCE = """
#define __host__
#define __device__
#define __forceinline__ inline
#include "%s/csrc/kernels/attn_deal.h"
// counts[s]: a sequence's units a head and row tile, and its row tiles with the heads; a read outside is noted in *bad
struct Counts { const unsigned *units, *tiles; int seqs, *bad; };
static unsigned read(const Counts &c, const unsigned *of, int s) {
  if (s < 0 || s >= c.seqs) { ++*c.bad; return 1; }
  return of[s];
}
// Workgroup `w`'s segments as (sequence, item of it, first unit, units, parts), at most `room`; the parts of whole items 1.
extern "C" int walk(const unsigned *summed_units, const unsigned *summed_tiles, const unsigned *units, const unsigned *tiles, int seqs, int w, int grid, int *out,
                    int room, int *bad) {
  Counts was{summed_units, summed_tiles, seqs, bad}, now{units, tiles, seqs, bad};
  unsigned total = 0, longest = 0;
  for (int s = 0; s < seqs; ++s) {
    const unsigned u = read(was, was.units, s), t = read(was, was.tiles, s);
    total += u * t;
    if (t && u > longest) longest = u;
  }
  if (!total) return 0;
  unsigned share = (total + grid - 1) / grid, least = (longest + AT_PARTS - 2) / (AT_PARTS - 1), base = 0;
  if (share < least) share = least;
  if ((unsigned)w > (total - 1) / share) return 0;
  unsigned at = w * share, last = at + share < total ? at + share : total, u = 0, t = 0;
  auto take = [&](int s) { u = read(now, units, s), t = read(now, tiles, s); };
  int s = at_walk([&](int i) { return take(i), u * t; }, 0, seqs, base, at);
  if (s >= seqs) return 0;
  unsigned it = (at - base) / u, u0 = at - base - it * u;
  for (int n = 0;;) {
    const unsigned u1 = u0 + (last - at) < u ? u0 + (last - at) : u, start = at - u0, first = start / share;
    if (n < room) {
      const int seg[] = {s, (int)it, (int)u0, (int)(u1 - u0), u0 == 0 && u1 == u ? 1 : at_parts_of(start, u, share, first, grid), (int)first};
      for (int i = 0; i < 6; ++i) out[6 * n + i] = seg[i];
    }
    ++n;
    at += u1 - u0, u0 = 0;
    if (at >= last) return n;
    if (++it == t) {
      it = 0;
      s = at_next([&](int i) { return take(i), t; }, s, seqs);
      if (s >= seqs) return n;
    }
  }
}
"""


@pytest.fixture(scope="module")
def walk(tmp_path_factory):
    at = tmp_path_factory.mktemp("deal")
    src, so = at / "walk.cpp", at / "walk.so"
    src.write_text(SOURCE % iu8.PKG)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", str(src), "-o", str(so)], check=True)
    lib = ctypes.CDLL(str(so))

    def call(summed, now, w, grid):
        arrays = [np.ascontiguousarray(x, np.uint32) for x in (*summed, *now)]
        out, bad = np.zeros((4096, 6), np.int32), ctypes.c_int(0)
        n = lib.walk(*(a.ctypes.data_as(ctypes.c_void_p) for a in arrays), len(arrays[0]), w, grid, out.ctypes.data_as(ctypes.c_void_p), len(out), ctypes.byref(bad))
        assert bad.value == 0, "a count outside the arrays was read"
        assert n <= len(out)
        return out[:n].tolist()

    return call


def test_every_unit_is_walked_once(walk):
    rng = np.random.default_rng(1)
    for _ in range(300):
        seqs, grid = int(rng.integers(1, 40)), int(rng.choice([3, 16, 128, 256]))
        units, tiles = rng.integers(1, 1 + rng.choice([2, 20, 900]), seqs), rng.integers(0, 4, seqs)
        seen = {(s, i): np.zeros(units[s], int) for s in range(seqs) for i in range(tiles[s])}
        parts = {}
        for w in range(grid):
            for s, it, u0, n, ns, first in walk((units, tiles), (units, tiles), w, grid):
                seen[s, it][u0:u0 + n] += 1
                parts.setdefault((s, it), []).append((w, ns, first))
        assert all((x == 1).all() for x in seen.values())
        for of in parts.values():          # all of an item's parts agree on how many there are, and whose slots they lie in
            assert {(ns, first) for _, ns, first in of} == {(len(of), of[0][0])} and len(of) <= 128


def test_counts_that_change_meanwhile_lead_out_of_no_array(walk):
    """Sequences released, begun, grown or shrunk between the sum and the walk: no count outside the arrays is read, and no join looks
    at slots that the grid does not have."""
    rng, moved = np.random.default_rng(2), 0
    for _ in range(600):
        seqs, grid = int(rng.integers(1, 40)), int(rng.choice([3, 16, 128, 256]))
        units, tiles = rng.integers(1, 1 + rng.choice([2, 20, 900]), seqs), rng.integers(0, 4, seqs)
        units_now, tiles_now = units.copy(), tiles.copy()
        for s in rng.integers(0, seqs, 1 + seqs // 3):
            units_now[s], tiles_now[s] = rng.choice([1, units[s], 5000]), rng.choice([0, tiles[s], 3])
        for w in range(grid):
            for s, it, u0, n, ns, first in walk((units, tiles), (units_now, tiles_now), w, grid):
                assert 0 <= s < seqs and 0 <= it < tiles_now[s] and 0 <= u0 < u0 + n <= units_now[s]
                assert 0 <= first and 1 <= ns <= 128 and first + ns <= grid
        moved += int((units_now * tiles_now).sum() < (units * tiles).sum())
    assert moved > 100          # walks that would otherwise have run on behind the last sequence


def test_all_sequences_released(walk):
    units, tiles = np.array([40, 3, 7]), np.array([2, 1, 4])
    none = np.zeros(3, int)
    assert all(walk((units, tiles), (np.ones(3, int), none), w, 16) == [] for w in range(16))
