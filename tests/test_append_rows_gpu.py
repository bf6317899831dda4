"""Appends of more than 512 rows, two a workgroup, whose last workgroup has one: contiguous caches against 64 bits, pages against
them, with the threads of few heads and of many; and equal rows that go to one page through many tables."""
import numpy as np
import pytest
import torch

import mingtts as mt
from _gpu_util import say
from _paged_util import TORCH
from test_kv_f8_gpu import INV, check_append, run_append

pytestmark = pytest.mark.gpu

CASES = [
    # B, T, hq, hkv, cap, pos, counts, offset
    (3, 171, 14, 2, 192, [0, 21, 30], None, 5),              # threads for both rows' heads
    (3, 171, 14, 2, 176, [0, 4, 100], [171, 170, 169], 0),    # ragged, the last row padding, slots past the cache
    (1, 513, 4, 1, 528, [9], None, 100000),                   # few heads
    (27, 19, 16, 16, 32, [b % 13 for b in range(27)], [19 - b % 3 for b in range(27)], 0),  # more heads than threads
]


@pytest.mark.parametrize("kind", ["f32", "f16", "f8"])
@pytest.mark.parametrize("case", CASES)
def test_odd_numbers_of_rows(gpu, kind, case):
    B, T, hq, hkv, cap, pos, counts, offset = case
    assert B * T > 512 and B * T % 2
    say(f"append {kind} {case[:5]}")
    qkv = np.random.default_rng(B + T).standard_normal((B * T, (hq + 2 * hkv) * 64)).astype(np.float32)
    kv, out = run_append(gpu, kind, *case, qkv)
    check_append(kv, out, kind, *case, qkv)
    # the same rows into pages
    n = cap // 16
    table = torch.randperm(B * n, generator=torch.Generator().manual_seed(T)).view(B, n).int().to(gpu)
    paged = mt.PagedKV.empty(B * n, hkv, 16, table, TORCH[kind])
    q = torch.full((B * T, hq * 64), -5.0, device=gpu)
    i = lambda a: None if a is None else torch.tensor(a, dtype=torch.int32, device=gpu)  # noqa: E731
    mt.rope_append_paged(torch.from_numpy(qkv).to(gpu), B, T, hq, hkv, i(pos), paged, torch.from_numpy(INV).to(gpu), q, counts=i(counts),
                         offset=offset)
    torch.cuda.synchronize()
    assert torch.equal(q, out[:B * T, :hq * 64])
    for b in range(B):
        slots = [pos[b] + t for t in range(T if counts is None else counts[b]) if pos[b] + t < cap]
        for name in ("k", "v") + (("k_scale", "v_scale") if kind == "f8" else ()):
            flat = getattr(paged, name)[table[b].long()].transpose(0, 1).flatten(1, 2)  # [hkv, cap, ...]
            assert torch.equal(flat[:, slots], getattr(kv, name)[b][:, slots]), (name, b)


@pytest.mark.parametrize("kind", ["f32", "f16", "f8"])
def test_equal_rows_through_two_entries(gpu, kind):
    """A prompt that every sequence appends for itself into the pages that all their tables name."""
    B, T, hq, hkv = 40, 30, 2, 2
    g = torch.Generator(device=gpu)
    g.manual_seed(1)
    one, inv = torch.randn(T, (hq + 2 * hkv) * 64, generator=g, device=gpu), torch.from_numpy(INV).to(gpu)
    kvs = [mt.PagedKV.empty(4, hkv, 16, torch.tensor([[2, 0]] * n, dtype=torch.int32, device=gpu), TORCH[kind]) for n in (1, B)]
    mt.rope_append_paged(one, 1, T, hq, hkv, None, kvs[0], inv)
    mt.rope_append_paged(one.repeat(B, 1), B, T, hq, hkv, None, kvs[1], inv)
    torch.cuda.synchronize()
    for name in ("k", "v") + (("k_scale", "v_scale") if kind == "f8" else ()):
        assert torch.equal(getattr(kvs[0], name), getattr(kvs[1], name)), name
