"""Caches that lie between each other: a sequence's keys, values and scales side by side in one allocation."""
import numpy as np
import pytest
import torch

import mingtts as mt
import _f8_util as U
from _gpu_util import say

pytestmark = pytest.mark.gpu
B, HKV, CAP = 3, 2, 24
INV = (1.0 / 1e6 ** (np.arange(32) / 32)).astype(np.float32)


def paired(gpu, dtype, fill):
    """k and v (and both scales) as the halves of one tensor, sequence by sequence."""
    c = torch.full((B, 2, HKV, CAP, 64), fill, dtype=dtype, device=gpu)
    if dtype != torch.uint8:
        return mt.KV(c[:, 0], c[:, 1])
    s = torch.full((B, 2, HKV, CAP), fill, dtype=dtype, device=gpu)
    return mt.KV(c[:, 0], c[:, 1], s[:, 0], s[:, 1])


def slabs(gpu, fill):
    """An 8-bit cache as one run of bytes a sequence: keys, values, then their scales."""
    n = HKV * CAP
    slab = torch.full((B, 130 * n), fill, dtype=torch.uint8, device=gpu)
    code = lambda at: slab[:, at:at + 64 * n].unflatten(1, (HKV, CAP, 64))  # noqa: E731
    scale = lambda at: slab[:, at:at + n].unflatten(1, (HKV, CAP))  # noqa: E731
    return mt.KV(code(0), code(64 * n), scale(128 * n), scale(129 * n))


def alike(a, b):
    return all(torch.equal(getattr(a, n), getattr(b, n)) for n in ("k", "v") + (("k_scale", "v_scale") if a.type == mt.F8 else ()))


LAYOUTS = [("f32", lambda g, f: paired(g, torch.float32, f)), ("f16", lambda g, f: paired(g, torch.float16, f)),
           ("f8", lambda g, f: paired(g, torch.uint8, f)), ("f8 slabs", slabs)]


@pytest.mark.parametrize("layout", LAYOUTS, ids=[n for n, _ in LAYOUTS])
def test_append_copy_and_attention(gpu, layout):
    name, make = layout
    say(f"interleaved {name}")
    rng = np.random.default_rng(1)
    qkv = torch.from_numpy(rng.standard_normal((B * 4, 18 * 64)).astype(np.float32)).to(gpu)
    pos = torch.tensor([0, 5, 20], dtype=torch.int32, device=gpu)
    inv = torch.from_numpy(INV).to(gpu)
    side = make(gpu, 1)
    dtype = side.k.dtype
    plain = mt.KV.empty(B, HKV, CAP, dtype, gpu)
    for n in ("k", "v"):
        getattr(plain, n).fill_(1)
    q = [torch.zeros(B * 4, 14 * 64, device=gpu) for _ in range(2)]
    out = [torch.zeros_like(q[0]) for _ in range(2)]
    for kv, a, o in ((side, q[0], out[0]), (plain, q[1], out[1])):
        mt.rope_append(qkv, B, 4, 14, HKV, pos, kv, inv, a)
        mt.attention_shared(a, B, 4, 14, HKV, pos, kv, o)
    assert alike(side, plain) and torch.equal(q[0], q[1]) and torch.equal(out[0], out[1])
    # from and into such caches, and between the halves of larger ones
    for src, dst in ((side, mt.KV.empty(B, HKV, CAP, dtype, gpu)), (plain, make(gpu, 0))):
        mt.kv_copy(src, dst, B, CAP)
        assert alike(src, dst)
    both = torch.zeros(B, 4, HKV, CAP, 64, dtype=torch.float16, device=gpu)
    low, high = mt.KV(both[:, 0], both[:, 1]), mt.KV(both[:, 2], both[:, 3])
    low.k.normal_()
    low.v.normal_()
    mt.kv_copy(low, high, B, CAP)
    assert alike(low, high)
