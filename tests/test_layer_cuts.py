"""The host's choice of the layers' tiles, asked of its own source: the sizes by which the products are tested take the tiles that they are
there for, and between them every one that a size can take."""
import ctypes
import os
import random
import subprocess

import pytest

from conftest import ROOT
from layer_tiles import FLOATS, HALVES, TILES

DTYPE = {HALVES: 2, FLOATS: 0}        # both 16-bit types are cut alike


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("cuts") / "layer_cuts.so")
    subprocess.run(["g++", "-O1", "-std=c++17", "-fPIC", "-shared", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), "-o", out,
                    os.path.join(ROOT, "tests", "layer_cuts.cpp")], check=True)
    return ctypes.CDLL(out)


def taken(lib, kind, what, rows, inner, outer):
    """(what, side, whether in parts, whether workgroups take several tiles) of one of the layer's products; None for few rows."""
    i64, out = ctypes.c_int64, (ctypes.c_int64 * 5)()
    across = None
    if what in ("forward", "codes"):
        lib.forward_cut(DTYPE[kind], i64(rows), i64(inner), i64(outer), what == "codes", 1, out)
        few, finished, side, parts = out[:4]
        if few:
            return None
        if finished:
            what = "finished"
        across, down, wide = -(-rows // side), outer, side
        if what == "codes":       # whole tiles of 256 columns, whatever the cut without codes would be
            parts, wide = 1, 256
    else:
        m, n, depth = (rows, inner, outer) if what == "dx" else (outer, inner, rows)
        lib.product_cut(DTYPE[kind], what == "dw", i64(m), i64(n), i64(depth), out)
        side, parts = out[:2]
        across, down, wide = -(-m // side), n, side
    slots = lib.compute_units() * (1 if what == "codes" else lib.workgroups_of_a_unit(side))
    return what, side, parts > 1, across * -(-down // wide) * parts > slots


@pytest.mark.parametrize("case", TILES, ids=str)
def test_the_sizes_take_their_tiles(lib, case):
    kind, what, side, parts, further, sizes = case
    # finished: parts, or codes that no tile holds
    got = taken(lib, kind, "codes" if what == "finished" else what, *sizes)
    assert got == (what, side, parts, further)


def test_every_tile_that_a_size_can_take_has_one(lib):
    rng = random.Random(3)
    size = lambda: rng.choice((rng.randint(8, 600), rng.randint(600, 3000), rng.randint(3000, 9000)))  # noqa: E731
    seen = set()
    for _ in range(60000):
        sizes = size(), size(), size()
        for kind in (HALVES, FLOATS):
            for what in ("forward", "codes", "dx", "dw"):
                t = taken(lib, kind, what, *sizes)
                # a plain forward product in parts runs through the same kernels as one with codes that are finished
                if t and not (what == "forward" and t[2]):
                    seen.add((kind,) + t)
    assert seen - {t[:5] for t in TILES} == set()
