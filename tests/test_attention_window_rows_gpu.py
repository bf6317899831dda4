"""mt_attention_paged and mt_attention_sinks over so many rows that workgroups share tiles of keys: every cache type, pages and
contiguous caches, windows and first positions, ragged and empty sequences, missing pages, values that are not finite.  A sample
of the rows is checked in 64 bits."""
import numpy as np
import pytest
import torch

from _gpu_util import say
from _paged_util import Case

pytestmark = pytest.mark.gpu
KINDS = ["f32", "f16", "f8"]


def sample(c, every=9):
    rng = np.random.default_rng(c.B)
    return {(b, t) for b in range(c.B) for t in range(c.T) if (b * c.T + t) % every == rng.integers(every) or t in (0, c.T - 1) and b < 3}


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page", [None, 16, 48, 128])
@pytest.mark.parametrize("B,T,hq,hkv,cap", [(64, 40, 14, 2, 100), (16, 100, 16, 16, 164), (3, 1400, 4, 2, 1500), (140, 20, 16, 1, 60)])
def test_many_rows(gpu, kind, page, B, T, hq, hkv, cap):
    say(f"many rows {kind} {page} {B} {T}")
    c = Case(gpu, kind, B, T, hq, hkv, cap, page=page)
    c.check(c.run(pad=8), rows=sample(c, 61 if T > 1000 else 29))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page", [None, 16, 64])
@pytest.mark.parametrize("window,sinks", [(1, 0), (5, 3), (64, 64), (65, 1), (100, 130), (10000, 2)])
def test_windows(gpu, kind, page, window, sinks):
    say(f"many rows, window {kind} {page} {window} {sinks}")
    c = Case(gpu, kind, 64, 40, 14, 2, 320, page=page, window=window, sinks=sinks)
    c.check(c.run(), rows=sample(c, 37))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page", [None, 32])
def test_ragged(gpu, kind, page):
    """Sequences of any number of rows, none among them, and rows past the cache."""
    B, T, cap = 64, 40, 96
    rng = np.random.default_rng(3)
    counts = [int(x) for x in rng.integers(0, T + 1, B)]
    counts[:3] = [0, T, 1]
    pos = [int(x) for x in rng.integers(0, cap, B)]
    pos[1] = 1000
    c = Case(gpu, kind, B, T, 14, 2, cap, page=page, pos=pos, counts=counts)
    c.check(c.run(), rows=sample(c, 11))


@pytest.mark.parametrize("kind", KINDS)
def test_missing_pages(gpu, kind):
    cap, page, B, T = 160, 16, 64, 40
    missing = [(b, (3 * b) % 10) for b in range(0, B, 2)] + [(7, e) for e in range(10)]
    c = Case(gpu, kind, B, T, 14, 2, cap, page=page, missing=missing)
    got = c.run()
    c.check(got, rows=sample(c, 23) | {(7, t) for t in range(T)})
    assert (got[7] == 0).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("scale,q_scale", [(0.125, 30.0), (-0.2, 3.0), (1.0, 1e-3), (1e-6, 1.0), (0.0, 1.0)])
def test_scales_of_the_scores(gpu, kind, scale, q_scale):
    c = Case(gpu, kind, 64, 40, 14, 2, 96, page=16, q_scale=q_scale)
    c.check(c.run(scale=scale), scale=scale, rows=sample(c, 31))


@pytest.mark.parametrize("kind", KINDS)
def test_scores_that_grow(gpu, kind):
    """Keys that get longer along the cache: the reference has to follow."""
    def values(i, x):
        if i == 0:
            x *= np.linspace(0.01, 12, x.shape[2], dtype=np.float32)[:, None]
    for B, T, cap in ((64, 40, 480), (2, 1, 480), (1, 1, 4000)):
        c = Case(gpu, kind, B, T, 14, 2, cap, page=16, values=values)
        c.check(c.run(), rows=sample(c, 41))


def test_blocks_of_very_different_sizes(gpu):
    def values(i, x):
        x *= 2.0 ** (np.random.default_rng(3 + i).integers(-15, 16, x.shape[:3] + (1,)) * (1.0 if i else 0.1))
    c = Case(gpu, "f8", 64, 40, 14, 2, 200, page=16, values=values)
    c.check(c.run(), rows=sample(c, 31))


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_values_that_are_not_finite(gpu, kind, bad):
    """A key or value that is not finite reaches the rows that attend it and no other."""
    B, T, cap, window = 64, 40, 120, 30
    for which in (0, 1):
        def values(i, x):
            if i == which:
                x[5, 1, 50, 3] = bad
        pos = [int(x) for x in np.random.default_rng(1).integers(0, 80, B)]
        pos[5] = 40
        c = Case(gpu, kind, B, T, 14, 2, cap, page=16, pos=pos, window=window, sinks=3, values=values)
        got = c.run()
        hit = [t for t in range(T) if 50 in c.keys(5, t)]
        assert 0 < len(hit) < T
        c.check(got, rows=(sample(c, 31) | {(5, t) for t in range(T)}) - {(5, t) for t in hit})
        assert np.isfinite(got[5, hit][:, :7]).all()  # the other key head
        for t in hit:
            for h in range(7, 14):
                if which == 1:
                    assert not np.isfinite(got[5, t, h, 3]) and np.isfinite(np.delete(got[5, t, h], 3)).all()
                elif c.q.reshape(B, T, 14, 64)[5, t, h, 3] * bad != -np.inf:
                    assert np.isnan(got[5, t, h]).all()
                else:
                    assert np.isfinite(got[5, t, h]).all()


def test_same_bits_in_any_layout_and_again(gpu):
    for kind in KINDS:
        out = []
        for page in (None, 16, 64):
            c = Case(gpu, kind, 64, 40, 14, 2, 320, page=page, window=100, sinks=20, seed=4)
            out.append(c.run())
        assert all((o == out[0]).all() for o in out[1:]) and (c.run() == out[0]).all()
