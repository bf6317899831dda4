"""Paged caches of more than 2^32 bytes: attention through every kernel, rows that are done again, and the append, with pages that
begin past 2^32 and no sequence's page where an offset cut to 32 bits would land."""
import numpy as np
import pytest
import torch

import mingtts as mt
from _gpu_util import say
from _paged_util import TORCH, Case
from _window_plan import plan_of
from test_append_paged_gpu import INV

pytestmark = pytest.mark.gpu
KINDS = ["f32", "f16", "f8"]
PAGE, HKV = 512, 2
CODE = 0x48  # what pages of no sequence hold, scales and codes alike: finite values unlike the rows'


def sample(c):
    rng = np.random.default_rng(c.B + c.T)
    return {(b, t) for b in range(c.B) for t in range(c.T) if rng.integers(60) == 0 or t in (0, c.T - 1)}


class Far:
    """A pool whose pages lie in one run of bytes, a page's keys, values and scales side by side, more than 2^32 bytes of it;
    the sequences' pages are among those that begin past 2^32.  The same bytes less 2^32 are pages of no sequence."""

    def __init__(self, gpu, kind, B, entries):
        es = torch.zeros(0, dtype=TORCH[kind]).element_size()
        each, scales = HKV * PAGE * 64 * es, HKV * PAGE
        step = 2 * each + 2 * scales
        self.first = 2 ** 32 // step + 1
        pages = self.first + 2 * B * entries + 5
        self.bytes = torch.full((pages * step,), CODE, dtype=torch.uint8, device=gpu)
        assert self.first * step >= 2 ** 32 and pages < 2 ** 32 * 2 // step  # (an offset less 2^32 is in the pool, and before `first`)
        flat = self.bytes.view(TORCH[kind])
        view = lambda at: flat.as_strided((pages, HKV, PAGE, 64), (step // es, PAGE * 64, 64, 1), at // es)  # noqa: E731
        byte = lambda at: self.bytes.as_strided((pages, HKV, PAGE), (step, PAGE, 1), at)  # noqa: E731
        table = self.first + np.random.default_rng(7).permutation(2 * B * entries)[:B * entries].reshape(B, entries)
        self.table = table.astype(np.int32)
        s = (byte(2 * each), byte(2 * each + scales)) if kind == "f8" else (None, None)
        self.kv = mt.PagedKV(view(0), view(each), torch.from_numpy(self.table).to(gpu), *s)

    def take(self, case):
        """The case's pages where this pool's table says."""
        for src, dst in zip(*([kv.k, kv.v] + ([kv.k_scale, kv.v_scale] if kv.k_scale is not None else []) for kv in (case.kv, self.kv))):
            for b in range(case.B):
                for e in range(case.table.shape[1]):
                    if case.table[b, e] >= 0:
                        dst[int(self.table[b, e])] = src[int(case.table[b, e])]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("B,T,hq,cap,window,plan", [
    (2, 3, 14, 1024, 200, "few"),
    (2, 20, 14, 400, 0, "few"),
    (2, 1, 14, 1500, 100, "few"),  # NaN in the window's first tile, before the window: rows are done again, each from its own keys
    (1, 1, 14, 4096, 0, "parts"),
    (2, 1060, 16, 1536, 0, "shared"),
    (2, 1060, 16, 1536, 333, "shared"),
])
def test_far_pages(gpu, kind, B, T, hq, cap, window, plan):
    say(f"far pages {kind} {B} {T} {cap} {window}")
    c = Case(gpu, kind, B, T, hq, HKV, cap, page=PAGE, pos=[cap - T, max(0, cap * 2 // 3 - T)][:B], window=window, sinks=window and 7)
    p = plan_of(c)
    assert plan == ("shared" if p.shared else "parts" if p.parts > 1 else "few")
    far = Far(gpu, kind, B, c.table.shape[1])
    far.take(c)
    c.check(c.run(kv=far.kv), rows=sample(c))


@pytest.mark.parametrize("kind", KINDS)
def test_append_into_far_pages(gpu, kind):
    """The rows of the same append into near pages, and no other byte."""
    B, T, hq, cap = 2, 40, 4, 1024
    far = Far(gpu, kind, B, cap // PAGE)
    near = mt.PagedKV.empty(B * 2, HKV, PAGE, torch.arange(B * 2, dtype=torch.int32, device=gpu).view(B, 2), TORCH[kind])
    g = torch.Generator(device=gpu)
    g.manual_seed(3)
    qkv = torch.randn(B * T, (hq + 2 * HKV) * 64, generator=g, device=gpu)
    pos, inv = torch.tensor([490, 30], dtype=torch.int32, device=gpu), torch.from_numpy(INV).to(gpu)
    for kv in (near, far.kv):
        mt.rope_append_paged(qkv, B, T, hq, HKV, pos, kv, inv)
    torch.cuda.synchronize()
    names = ("k", "v") + (("k_scale", "v_scale") if kind == "f8" else ())
    for b, p0 in enumerate((490, 30)):
        for p in range(p0, p0 + T):
            for n in names:
                a, z = (getattr(kv, n)[int(kv.table[b, p // PAGE]), :, p % PAGE] for kv in (near, far.kv))
                assert torch.equal(a, z), (n, b, p)
                z.view(torch.uint8).fill_(CODE)
    assert bool((far.bytes == CODE).all())
