"""The placement of attention over pages and windows without a GPU: which shapes of workgroups the rule can choose, and the
workspace that a call without a bound of its length needs."""
import random
import re

import pytest

import mingtts as mt
from _window_plan import window_plan
from test_paged_abi import attend, contiguous, paged

TYPES = [mt.F32, mt.F16, mt.F8]


@pytest.mark.parametrize("t", TYPES)
def test_shapes_of_workgroups(t):
    """Rows that share tiles in LDS take four waves of 16 rows; other workgroups' waves share one row tile, or two where there
    are four waves and the keys are not split.  The kernels are compiled for these alone."""
    rng = random.Random(t)
    seen = set()
    for _ in range(60000):
        hkv, G = rng.choice([1, 1, 2, 2, 4, 8, 16, 32]), rng.choice([1, 2, 3, 4, 6, 7, 8, 12, 16, 32, 100])
        B, T, n = (int(2 ** rng.uniform(0, top)) for top in (12, 13, 20))
        window, sinks = rng.choice([0, int(2 ** rng.uniform(0, 14))]), rng.choice([0, int(2 ** rng.uniform(0, 10))])
        p = window_plan(B, T, G * hkv, hkv, n, window, sinks, t)
        seen.add((p.shared, p.waves, p.keys, p.parts > 1))
        if p.parts > 1:
            tk = 32 if t == mt.F32 else 64
            own = max(1, min(n, window + sinks + T - 1 if window else n))
            assert p.run > 0 and (p.parts - 1) * p.run < -(-own // tk) <= p.parts * p.run
        else:
            assert p.parts == 1
    assert seen == {(True, 4, 1, False), (False, 4, 2, False), (False, 4, 4, False), (False, 8, 8, False), (False, 4, 4, True), (False, 8, 8, True)}


@pytest.mark.parametrize("make", [paged, contiguous])
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("window,sinks", [(0, 0), (50000, 100)])
def test_workspace_without_a_bound(make, t, window, sinks):
    """A call with len_max 0 needs the workspace that is asked for with the number of slots."""
    kv = make(t=t, table_len=8192, table_stride=8192, pages=8192) if make is paged else make(t=t, cache_len=1 << 17)
    need = mt.load().mt_attention_window_workspace(1, 1, 14, 2, 1 << 17, window, sinks, t)
    assert need > 0
    assert attend(kv, B=1, window=window, sinks=sinks) == mt.EINVAL
    assert int(re.search(r"needs (\d+) bytes", mt.last_error()).group(1)) == need
    assert attend(kv, B=1, window=window, sinks=sinks, ws=1 << 50, wsn=need - 1) == mt.EINVAL
    assert "needs" in mt.last_error()


def test_workspace_of_no_key_is_none():
    """0 is no way to ask for all slots: the query does not know the caches."""
    assert mt.load().mt_attention_window_workspace(1, 1, 14, 2, 0, 0, 0, mt.F16) == 0
