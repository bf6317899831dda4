"""mt_attention_paged and mt_attention_sinks against 64 bits, row by row: every cache type, pages of all kinds of sizes and
contiguous caches, windows with first positions that stay visible, ragged rows, head layouts, slots past the cache,
slots and pages that a row must not see."""
import numpy as np
import pytest
import torch

import mingtts as mt
from _gpu_util import say
from _paged_util import Case, poison, to_pages

pytestmark = pytest.mark.gpu
KINDS = ["f32", "f16", "f8"]

SHAPES = [
    # B, T, hq, hkv, cap
    (1, 1, 1, 1, 4),
    (2, 1, 14, 2, 512),
    (1, 1, 14, 2, 40),
    (5, 1, 16, 16, 132),
    (3, 1, 16, 1, 260),
    (40, 1, 8, 2, 64),
    (2, 1, 40, 2, 72),
    (1, 1, 14, 2, 5000),
    (2, 9, 14, 2, 64),
    (3, 17, 12, 4, 48),
    (2, 50, 14, 2, 100),
    (1, 130, 4, 1, 200),
    (2, 300, 14, 2, 420),
]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page", [None, 16, 48])
@pytest.mark.parametrize("shape", SHAPES)
def test_attention(gpu, kind, page, shape):
    say(f"attention {kind} {page} {shape}")
    c = Case(gpu, kind, *shape, page=page)
    c.check(c.run(pad=4), rows=None if shape[0] * shape[1] < 400 else {(b, t) for b in range(2) for t in range(0, 300, 7)})


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page", [16, 32, 80, 256, 1024])
def test_page_sizes(gpu, kind, page):
    say(f"pages of {page} {kind}")
    for T in (1, 40):
        c = Case(gpu, kind, 3, T, 14, 2, 700, page=page)
        c.check(c.run())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page", [None, 16])
@pytest.mark.parametrize("B,T,pos,counts", [
    (4, 1, [0, 0, 63, 62], None),
    (4, 1, [0, 31, 32, 33], [1, 0, 1, 1]),
    (3, 6, [0, 58, 20], [1, 6, 0]),
    (3, 6, [60, 64, 1000], [6, 2, 1]),  # rows past the cache attend all of it
    (2, 1, [2 ** 31 - 1, -1], None),
    (2, 40, [0, 24], [33, 40]),
    (1, 150, [0], [149]),
])
def test_ragged(gpu, kind, page, B, T, pos, counts):
    say(f"ragged {kind} {page} {B} {T}")
    c = Case(gpu, kind, B, T, 14, 2, 64 if T < 100 else 160, page=page, pos=[p % 2 ** 32 for p in pos], counts=counts)
    c.pos = [p - 2 ** 32 if p >= 2 ** 31 else p for p in c.pos]
    got = c.run()
    c.pos = [p % 2 ** 32 for p in pos]
    c.check(got)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page", [None, 16, 64])
@pytest.mark.parametrize("window", [1, 5, 64, 65, 200, 10000])
@pytest.mark.parametrize("sinks", [0, 1, 16, 70, 1000])
def test_window_and_sinks(gpu, kind, page, window, sinks):
    say(f"window {kind} {page} {window} {sinks}")
    for B, T, cap in ((3, 1, 300), (2, 20, 292), (1, 140, 384)):
        c = Case(gpu, kind, B, T, 14, 2, cap, page=page, window=window, sinks=sinks)
        c.check(c.run())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page", [None, 256])
def test_long_split_and_hints(gpu, kind, page):
    """Few rows over many keys, and bounds of the length that are too small, exact and too large."""
    c = Case(gpu, kind, 2, 1, 14, 2, 20000, page=page, pos=[19999, 12345])
    for len_max in (0, 1, 700, 20000, 2 ** 31):
        c.check(c.run(len_max=len_max))
    c = Case(gpu, kind, 3, 2, 8, 2, 9000, page=page, pos=[8998, 17, 4000], counts=[2, 1, 2], window=3000, sinks=2100)
    for len_max in (0, 40, 9000):
        c.check(c.run(len_max=len_max))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("B,T,hq,hkv,cap", [
    (1, 1, 4, 1, 512), (3, 1, 4, 1, 700), (1, 1, 14, 2, 1600), (2, 3, 4, 2, 3000), (8, 1, 2, 1, 8192), (1, 1, 7, 1, 33000),
    (33, 1, 2, 1, 2100), (40, 1, 4, 2, 1000), (70, 1, 2, 2, 2600), (150, 1, 1, 1, 2052), (5, 20, 2, 1, 1700),
])
def test_parts_of_many_sizes(gpu, kind, B, T, hq, hkv, cap):
    """Keys split into few and many parts, of four waves and of eight, the last part shorter, sequences that end in the first."""
    say(f"parts {kind} {B} {T} {cap}")
    pos = [(cap - T, 5, cap // 2, 130)[b % 4] for b in range(B)]
    c = Case(gpu, kind, B, T, hq, hkv, cap, page=64, pos=pos)
    c.check(c.run(), rows={(b, t) for b in range(min(B, 12)) for t in range(T)})


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page", [None, 32])
@pytest.mark.parametrize("T", [1, 30])
@pytest.mark.parametrize("scale,q_scale", [(0.125, 30.0), (-0.2, 3.0), (1.0, 1e-3), (1e-6, 1.0), (0.0, 1.0)])
def test_scales_of_the_scores(gpu, kind, page, T, scale, q_scale):
    c = Case(gpu, kind, 3, T, 14, 2, 96, page=page, q_scale=q_scale)
    c.check(c.run(scale=scale), scale=scale)


@pytest.mark.parametrize("T", [1, 140])
def test_blocks_of_very_different_sizes(gpu, T):
    """8-bit values whose scales lie 2^30 apart from key to key."""
    def values(i, x):
        if i == 1:
            x *= 2.0 ** np.random.default_rng(3).integers(-15, 16, x.shape[:3] + (1,))
    c = Case(gpu, "f8", 2, T, 14, 2, 200, page=16, values=values)
    c.check(c.run())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T", [1, 33, 140])
def test_missing_pages(gpu, kind, T):
    """Slots without a page weigh nothing; rows without any page are zeros."""
    cap, page = 320, 16
    c = Case(gpu, kind, 3, T, 14, 2, cap, page=page, pos=[cap - T, 100, 0],
             missing=[(0, 3), (0, 7), (1, 0), (1, 6)] + [(2, e) for e in range(cap // page)])
    got = c.run()
    c.check(got)
    assert (got[2] == 0).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page", [None, 16])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_values_that_are_not_finite(gpu, kind, page, bad):
    """A key or value that is not finite reaches the rows that attend it and no other."""
    if kind == "f8" and not np.isnan(bad):
        pytest.skip("8 bits hold NaN only")
    B, T, hq, hkv, cap, window = 1, 140, 4, 2, 200, 30
    for which in (0, 1):
        def values(i, x):
            if i == which:
                x[0, 1, 100, 3] = bad
        c = Case(gpu, kind, B, T, hq, hkv, cap, page=page, pos=[40], window=window, sinks=3, values=values)
        got = c.run()
        hit = [t for t in range(T) if 100 in c.keys(0, t)]
        clean = {(0, t) for t in range(T)} - {(0, t) for t in hit}
        c.check(got, rows=clean)
        assert np.isfinite(got[0, hit][:, :2]).all()  # the other key head
        for t in hit:
            for h in (2, 3):
                if which == 1:  # the value's dim, and no other
                    assert not np.isfinite(got[0, t, h, 3]) and np.isfinite(np.delete(got[0, t, h], 3)).all()
                    continue
                s = c.q.reshape(T, hq, 64)[t, h, 3] * bad
                if s == -np.inf:  # no weight
                    j = c.keys(0, t)
                    j = j[j != 100]
                    w = np.exp((c.val[0][0, 1, j] @ c.q.reshape(T, hq, 64)[t, h].astype(np.float64)) * 0.125)
                    assert np.abs(got[0, t, h] - w @ c.val[1][0, 1, j] / w.sum()).max() < 1e-4
                else:
                    assert np.isnan(got[0, t, h]).all()


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("page", [None, 16])
def test_rows_of_scores_without_weight(gpu, kind, page):
    """Scores of -infinity alone: zeros, as for a row without a key."""
    def values(i, x):
        if i == 0:
            x[0, 0, :, 0] = -np.inf
    c = Case(gpu, kind, 2, 1, 2, 1, 96, page=page, pos=[80, 80], values=values)
    c.q[:, 0::64] = 1.0
    got = c.run()
    assert (got[0] == 0).all()
    c.check(got, rows={(1, 0)})


def test_far_pages(gpu):
    """A pool past 2^32 bytes: offsets of 64 bits."""
    page, hkv, pool = 512, 2, 40000
    k = torch.zeros(pool, hkv, page, 64, dtype=torch.uint8, device=gpu)
    assert k.numel() > 2 ** 31
    v, ks, vs = torch.zeros_like(k), torch.ones(pool, hkv, page, dtype=torch.uint8, device=gpu), torch.ones(pool, hkv, page, dtype=torch.uint8, device=gpu)
    c = Case(gpu, "f8", 2, 3, 14, 2, 1024, page=page, pos=[1021, 600])
    far = np.array([[pool - 1, 36000], [33333, pool - 2]], np.int32)
    near = c.kv
    for src, dst in ((near.k, k), (near.v, v), (near.k_scale, ks), (near.v_scale, vs)):
        for b in range(2):
            for e in range(2):
                if c.table[b, e] >= 0:
                    dst[int(far[b, e])] = src[int(c.table[b, e])]
    c.check(c.run(kv=mt.PagedKV(k, v, torch.from_numpy(far).to(gpu), ks, vs)))


@pytest.mark.parametrize("kind", KINDS)
def test_strided_pools_and_tables(gpu, kind):
    """Keys and values side by side in one pool, a table that is part of a larger one, a pool of a single page."""
    c = Case(gpu, kind, 3, 1, 14, 2, 256, page=32)
    k, v = c.kv.k, c.kv.v
    both = torch.stack([k, v], 1)
    scales = torch.stack([c.kv.k_scale, c.kv.v_scale], 1) if kind == "f8" else None
    wide = torch.full((5, 20), -1, dtype=torch.int32, device=gpu)
    wide[1:4, 3:11] = torch.from_numpy(c.table).to(gpu)
    s = (None, None) if scales is None else (scales[:, 0], scales[:, 1])
    c.check(c.run(kv=mt.PagedKV(both[:, 0], both[:, 1], wide[1:4, 3:11], *s)))
    c = Case(gpu, kind, 1, 2, 14, 2, 32, page=32)
    p = int(c.table[0, 0])
    one = [None if x is None else x[p:p + 1] for x in (c.kv.k, c.kv.v, c.kv.k_scale, c.kv.v_scale)]
    c.check(c.run(kv=mt.PagedKV(one[0], one[1], torch.zeros(1, 1, dtype=torch.int32, device=gpu), *one[2:])))


def test_shared_pages(gpu):
    """Many sequences whose tables begin with the same pages, as behind one prompt."""
    B, cap, page = 6, 160, 16
    c = Case(gpu, "f16", B, 1, 14, 2, cap, page=page, pos=[100 + 7 * b for b in range(B)])
    for x in c.val:
        x[:, :, :64] = x[:1, :, :64]
    c.table[:, :4] = c.table[0, :4]
    c.kv.table.copy_(torch.from_numpy(c.table))
    c.check(c.run())


@pytest.mark.parametrize("page", [None, 64])
def test_same_bits_again_and_on_another_stream(gpu, page):
    c = Case(gpu, "f16", 2, 1, 14, 2, 9000, page=page, pos=[8999, 5000])
    first = c.run()
    assert (c.run() == first).all()
    s = torch.cuda.Stream()
    assert (c.run(stream=s) == first).all()
    need = mt.load().mt_attention_window_workspace(2, 1, 14, 2, 9000 if page is None else 9024, 0, 0, mt.F16)
    ws = torch.full((max(need, 16),), 0xFF, dtype=torch.uint8, device=gpu)
    for _ in range(2):
        assert (c.run(workspace=ws) == first).all()
