"""mt_rope_append_paged: the bits of mt_rope_append in the table's pages, every type and page size; slots past the table and
without a page; rows and pages that stay as they were."""
import numpy as np
import pytest
import torch

import mingtts as mt
import _f8_util as U
from _gpu_util import say
from _paged_util import TORCH

pytestmark = pytest.mark.gpu
INV = (1.0 / 1e6 ** (np.arange(32) / 32)).astype(np.float32)


def filled(kind, shape, gpu):
    return torch.full(shape, 7, dtype=TORCH[kind], device=gpu)


@pytest.mark.parametrize("kind", ["f32", "f16", "f8"])
@pytest.mark.parametrize("B,T,hq,hkv,page,entries", [(2, 1, 14, 2, 16, 4), (3, 9, 8, 2, 32, 2), (1, 1, 1, 1, 16, 1), (300, 2, 16, 16, 16, 2),
                                                     (4, 70, 12, 4, 48, 3), (2, 5, 0, 3, 1024, 1)])
def test_append(gpu, kind, B, T, hq, hkv, page, entries):
    say(f"append {kind} {B} {T} {page}")
    rng = np.random.default_rng(B * T + page)
    cap, pool = page * entries, B * entries + 2
    # any slot, some rows past the table's last
    pos = torch.tensor(rng.integers(0, cap, B), dtype=torch.int32, device=gpu)
    counts = torch.tensor(rng.integers(0, T + 1, B), dtype=torch.int32, device=gpu)
    qkv = torch.from_numpy(rng.standard_normal((B * T, (hq + 2 * hkv) * 64)).astype(np.float32)).to(gpu)
    inv = torch.from_numpy(INV).to(gpu)
    table = torch.from_numpy(rng.permutation(pool)[:B * entries].reshape(B, entries).astype(np.int32)).to(gpu)
    table[0, entries - 1] = -1
    if B > 2:
        table[2, 0] = pool
    shape = (pool, hkv, page)
    scales = [filled("f8", shape, gpu) for _ in range(2)] if kind == "f8" else [None, None]
    kv = mt.PagedKV(filled(kind, shape + (64,), gpu), filled(kind, shape + (64,), gpu), table, *scales)
    flat = (B, hkv, cap)
    fs = [filled("f8", flat, gpu) for _ in range(2)] if kind == "f8" else [None, None]
    ref = mt.KV(filled(kind, flat + (64,), gpu), filled(kind, flat + (64,), gpu), *fs)
    q, q_ref = (torch.full((B * T, hq * 64), -3.0, device=gpu) for _ in range(2))
    mt.rope_append(qkv, B, T, hq, hkv, pos, ref, inv, q_ref if hq else None, counts=counts, offset=100000)
    mt.rope_append_paged(qkv, B, T, hq, hkv, pos, kv, inv, q if hq else None, counts=counts, offset=100000)
    torch.cuda.synchronize()
    assert torch.equal(q, q_ref)
    tab = table.cpu().numpy()
    for name in ("k", "v") + (("k_scale", "v_scale") if kind == "f8" else ()):
        got, want = getattr(kv, name), getattr(ref, name)
        left = torch.ones(pool, dtype=torch.bool, device=gpu)
        for b in range(B):
            for e in range(entries):
                if 0 <= tab[b, e] < pool:
                    assert torch.equal(got[tab[b, e]], want[b, :, e * page:(e + 1) * page]), (name, b, e)
                    left[tab[b, e]] = False
        assert (got[left] == 7).all()


def test_against_64_bits(gpu):
    """The rotation and the rounding themselves, at a far position."""
    B, T, hq, hkv, page, offset = 1, 3, 4, 2, 16, 2 ** 20
    x = np.random.default_rng(5).standard_normal((T, hq + 2 * hkv, 64)).astype(np.float32)
    table = torch.tensor([[4, 0]], dtype=torch.int32, device=gpu)
    q = torch.zeros(T, hq * 64, device=gpu)
    for kind in ("f32", "f16"):
        kv = mt.PagedKV.empty(5, hkv, page, table, TORCH[kind])
        mt.rope_append_paged(torch.from_numpy(x.reshape(T, -1)).to(gpu), B, T, hq, hkv, torch.tensor([14], dtype=torch.int32, device=gpu),
                             kv, torch.from_numpy(INV).to(gpu), q, offset=offset)
        torch.cuda.synchronize()
        for t in range(T):
            p = 14 + t
            rot = U.rope64(x[t, :hq + hkv].astype(np.float64), offset + p, INV)
            at = (int([4, 0][p // page]), slice(None), p % page)
            k, v = (getattr(kv, n)[at].cpu().double().numpy() for n in ("k", "v"))
            half = 2.0 ** -24 if kind == "f32" else 2.0 ** -11
            # half a step of the value, and 2^-50 or so of the pair for the rotation in 64 bits
            assert (np.abs(q.cpu().double().numpy().reshape(T, hq, 64)[t] - rot[:hq]) <= 2.0 ** -24 * np.abs(rot[:hq]) + 1e-14).all()
            assert (np.abs(k - rot[hq:]) <= half * np.abs(rot[hq:]) + 2.0 ** -25 * (kind == "f16") + 1e-14).all()
            assert (np.abs(v - x[t, hq + hkv:]) <= half * np.abs(x[t, hq + hkv:]) + 2.0 ** -25 * (kind == "f16")).all()


def test_in_place(gpu):
    """q = qkv at the same stride: the query heads rotated where they stand, keys and values as they were."""
    B, T, hq, hkv = 2, 3, 4, 1
    g = torch.Generator(device=gpu)
    g.manual_seed(1)
    qkv = torch.randn(B * T, (hq + 2 * hkv) * 64, generator=g, device=gpu)
    inv = torch.from_numpy(INV).to(gpu)
    table = torch.tensor([[1], [0]], dtype=torch.int32, device=gpu)
    kv, kv2 = (mt.PagedKV.empty(2, hkv, 16, table, torch.float16) for _ in range(2))
    q, both = torch.zeros(B * T, hq * 64, device=gpu), qkv.clone()
    mt.rope_append_paged(qkv, B, T, hq, hkv, None, kv, inv, q)
    mt.rope_append_paged(both, B, T, hq, hkv, None, kv2, inv, both)
    torch.cuda.synchronize()
    assert torch.equal(both[:, :hq * 64], q) and torch.equal(both[:, hq * 64:], qkv[:, hq * 64:])
    assert torch.equal(kv.k, kv2.k) and torch.equal(kv.v, kv2.v)
