"""Paths of mt_attention_paged and mt_attention_sinks that only some sizes take, each case checked against the placement that it
is for: two row tiles a workgroup, tiles and tables so long that a wave's places are made anew."""
import numpy as np
import pytest

from _gpu_util import say
from _paged_util import Case
from _window_plan import plan_of

pytestmark = pytest.mark.gpu
KINDS = ["f32", "f16", "f8"]


def sample(c, every, always=()):
    rng = np.random.default_rng(c.B + c.T)
    n = [c.T] * c.B if c.counts is None else c.counts
    rows = {(b, t) for b in range(c.B) for t in range(n[b]) if rng.integers(every) == 0 or t in (0, n[b] - 1)}
    return rows | set(always)


# ------------------------------------------------- two row tiles a workgroup --

def two_tiles(gpu, kind, page, **o):
    """Four heads a key head: a row tile is four tokens, a workgroup eight.  Sequences end in a workgroup's first tile, at its
    end, in the second, and in the next workgroup."""
    B, T = 75, 16
    counts = [0, 16, 1, 3, 4, 5, 7, 8, 9, 12, 13, 15] + [int(n) for n in np.random.default_rng(1).integers(0, T + 1, B - 12)]
    c = Case(gpu, kind, B, T, 16, 4, 448, page=page, counts=counts, **o)
    p = plan_of(c)
    assert (p.shared, p.waves, p.keys, p.parts) == (False, 4, 2, 1)
    return c


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page", [None, 16, 64])
@pytest.mark.parametrize("window,sinks", [(0, 0), (90, 20), (5, 0)])
def test_two_row_tiles(gpu, kind, page, window, sinks):
    say(f"two row tiles {kind} {page} {window}")
    c = two_tiles(gpu, kind, page, window=window, sinks=sinks)
    c.check(c.run(pad=4), rows=sample(c, 4, {(b, t) for b in range(12) for t in range(16)}))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page", [None, 16])
def test_two_row_tiles_and_a_value_that_is_not_finite(gpu, kind, page):
    """It reaches the rows from its slot on, in the workgroup's second tile, and no row before them."""
    pos = [int(p) for p in np.random.default_rng(2).integers(0, 430, 75)]
    pos[1] = 200

    def values(i, x):
        if i == 1:
            x[1, 2, 206, 9] = np.nan
    c = two_tiles(gpu, kind, page, pos=pos, values=values)
    got = c.run()
    c.check(got, rows=sample(c, 4) - {(1, t) for t in range(6, 16)} | {(1, t) for t in range(6)})
    bad = np.isnan(got[1])
    want = np.zeros_like(bad)
    want[6:, 8:12, 9 if kind != "f8" else slice(None)] = True
    if kind == "f8":  # (a block with a NaN: the codes that hold it, as the decoded values say)
        want[6:, 8:12] = np.isnan(c.val[1][1, 2, 206])
    assert (bad == want).all()


# ------------------------------------------------ places made anew on the way --

@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page", [None, 16, 48])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1500, 100)])
def test_long_shared_tiles(gpu, kind, page, window, sinks):
    """Workgroups that share tiles over more of them (16 of 64 keys, 32 of 32) than a wave holds the places of; missing pages before
    and after that."""
    say(f"long shared tiles {kind} {page} {window}")
    missing = [(0, s // page) for s in (5, 333, 1050, 1100, 1500, 2048)] if page else []
    c = Case(gpu, kind, 1, 2080, 16, 1, 2100, page=page, pos=[20], window=window, sinks=sinks, missing=missing)
    assert plan_of(c).shared
    c.check(c.run(), rows=sample(c, 150, {(0, t) for t in (1003, 1004, 1005, 1028, 1480, 1900, 2027, 2028, 2029)}))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page", [None, 16])
def test_long_shared_tiles_by_xcd(gpu, kind, page):
    c = Case(gpu, kind, 2, 2050, 8, 8, 2080, page=page, pos=[30, 0], counts=[2050, 1999],
             missing=[(0, 7), (0, 70), (1, 124)] if page else [])
    p = plan_of(c)
    assert p.shared and p.by_xcd
    c.check(c.run(), rows=sample(c, 150))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page", [None, 16, 32, 48, 64])
@pytest.mark.parametrize("window,sinks", [(0, 0), (4700, 60)])
def test_long_tables_of_few_rows(gpu, kind, page, window, sinks):
    """A wave's 16 tiles or more (as few as a wave holds the places of in pages that do not hold whole tiles); the bound of the
    length keeps the keys from being split."""
    say(f"long tables {kind} {page} {window}")
    missing = [(0, s // page) for s in (100, 4090, 4200, 4992)] + [(1, s // page) for s in (0, 4097, 4500)] if page else []
    c = Case(gpu, kind, 2, 1, 14, 2, 5000, page=page, pos=[4999, 4600], window=window, sinks=sinks, missing=missing)
    p, tk = plan_of(c, 1), 32 if kind == "f32" else 64
    assert not p.shared and p.parts == 1 and 5000 // tk // p.keys > 1024 // tk
    c.check(c.run(len_max=1))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page", [None, 16, 48])
def test_long_tables_of_many_row_tiles(gpu, kind, page):
    c = Case(gpu, kind, 1, 4830, 1, 1, 4900, page=page, pos=[60], missing=[(0, s // page) for s in (9, 2222, 4100, 4444, 4888)] if page else [])
    p = plan_of(c)
    assert (p.shared, p.waves, p.keys, p.parts) == (False, 4, 4, 1)
    c.check(c.run(), rows=sample(c, 200, {(0, t) for t in range(4036, 4050)}))
