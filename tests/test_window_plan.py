"""The placement of attention over pages and windows without a GPU: which shapes of workgroups the rule can choose."""
import random

import pytest

import mingtts as mt
from _window_plan import window_plan

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
