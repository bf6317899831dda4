"""mt_attention_shared where scores of attended keys are NaN: the row is NaN, wherever its keys are placed (one pass, parts
joined by a second kernel, a row done again alone) and however many of them stand together; a -infinity is no weight."""
import numpy as np
import pytest
import torch

import mingtts as mt
import _f8_util as U
from _gpu_util import say
from test_attention_shared_gpu import Case

pytestmark = pytest.mark.gpu
KINDS = ["f32", "f16", "f8"]


def spoil(c, part, where):
    """NaN keys at an index of a cache."""
    part[0][0][where] = 127 if c.kind == "f8" else float("nan")


def workspace(c):
    return mt.load().mt_attention_shared_workspace(c.B, c.T, c.hq, c.hkv, c.P, c.cap, 0, {"f32": mt.F32, "f16": mt.F16, "f8": mt.F8}[c.kind])


def rows_agree(c, got, nan, clean):
    """Rows of `nan` ([B, T, hq] truth values) are NaN throughout, the others what they were."""
    assert np.isnan(got[nan]).all(), "a NaN was lost"
    for b, t, h in np.argwhere(~nan):
        want, tol = c.want(b, t, h)
        assert np.abs(got[b, t, h] - want).max() <= tol and np.abs(clean[b, t, h] - want).max() <= tol


@pytest.mark.parametrize("kind", KINDS)
def test_the_only_own_key_of_a_split_row(gpu, kind):
    say(f"own key {kind}")
    c = Case(gpu, kind, 16, 1, 14, 2, 512, 8192, pos=[511, 3, 70, 0] + [200] * 12)
    assert workspace(c) > 0  # prefix and own keys in parts of their own
    clean = c.run()
    spoil(c, c.own, (3, 0, 0))
    nan = np.zeros((16, 1, 14), bool)
    nan[3, 0, :7] = True
    rows_agree(c, c.run(), nan, clean)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("keys", [slice(0, 8192), slice(0, 4096), slice(4096, 8192), slice(5000, 5001)])
def test_keys_of_the_prefix(gpu, kind, keys):
    say(f"prefix keys {kind} {keys}")
    c = Case(gpu, kind, 3, 1, 14, 2, 64, 8192, pos=[63, 0, 20])
    assert workspace(c) > 0
    clean = c.run()
    spoil(c, c.pre, (1, keys))
    nan = np.zeros((3, 1, 14), bool)
    nan[:, :, 7:] = True
    rows_agree(c, c.run(), nan, clean)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("lo,hi", [(0, 64), (0, 128), (64, 300), (0, 301), (300, 301)])
def test_keys_in_one_pass(gpu, kind, lo, hi):
    """Whole blocks of 64 keys, the first ones among them, and rows of nothing else."""
    say(f"one pass {kind} {lo} {hi}")
    c = Case(gpu, kind, 2, 1, 14, 2, 512, 0, pos=[300, 400])
    assert workspace(c) == 0
    clean = c.run()
    spoil(c, c.own, (0, 0, slice(lo, hi)))
    nan = np.zeros((2, 1, 14), bool)
    nan[0, 0, :7] = True
    rows_agree(c, c.run(), nan, clean)


@pytest.mark.parametrize("kind", KINDS)
def test_keys_of_prompts(gpu, kind):
    """Row tiles over four waves: a NaN key reaches its own row and the later ones only."""
    say(f"prompts {kind}")
    c = Case(gpu, kind, 9, 70, 8, 8, 80, 200, pos=[0] * 9, counts=[70, 5] + [40] * 7)
    clean = c.run()
    spoil(c, c.own, (0, 2, 64))
    nan = np.zeros((9, 70, 8), bool)
    nan[0, 64:, 2] = True
    got = c.run()
    assert np.isnan(got[nan]).all() and not np.isnan(got[~nan]).any()
    got[nan] = clean[nan]
    c.check(got)


@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_minus_infinity_over_a_whole_part(gpu, kind):
    """Keys whose scores are -infinity weigh nothing, a whole part of them too."""
    say(f"minus infinity {kind}")
    c = Case(gpu, kind, 2, 1, 14, 2, 64, 8192, pos=[63, 20])
    assert workspace(c) > 0
    c.q.reshape(2, 14, 64)[..., 0] = 1.0
    c.pre[0][0][1, :6000, 0] = -float("inf")
    got = c.run()
    for b in range(2):
        for h in range(14):
            kh, n = h // 7, c.pos[b] + 1
            first = 6000 if kh else 0
            kk, vv = (np.concatenate([p[2][kh, first:8192], o[2][b, kh, :n]]) for p, o in zip(c.pre, c.own))
            want, tol = U.attend64(c.q.reshape(2, 14, 64)[b, h].astype(np.float64), kk, vv, 0, len(kk), 0.125)
            assert np.abs(got[b, 0, h] - want).max() <= tol


@pytest.mark.parametrize("kind", KINDS)
def test_a_scale_of_zero(gpu, kind):
    """All weights alike, in parts with windows that leave some of them empty."""
    c = Case(gpu, kind, 40, 1, 14, 2, 512, 8192)
    for window in (0, 5000, 40):
        c.check(c.run(scale=0.0, window=window), scale=0.0, window=window)
