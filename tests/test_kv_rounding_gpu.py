"""mt_rope_append to the last bit: what is written is the rounding of the 64-bit rotation."""
import numpy as np
import pytest
import torch

import mingtts as mt
import _f8_util as U
from _gpu_util import say

pytestmark = pytest.mark.gpu
INV = (1.0 / 1e6 ** (np.arange(32) / 32)).astype(np.float32)
T, OFFSET = 4096, 9000
# The 64-bit angles are below 2^14: off by 2^-53 of that in each of the two computations, and a few such steps in sine, cosine
# and the rotation: under 1e-11 of |x0| + |x1|.
SLACK = 1e-11


def appended(gpu, kind):
    """T rows of one sequence in a cache of a type; q, the cache and the rotation in 64 bits with its slack."""
    rng = np.random.default_rng(12)
    qkv = rng.standard_normal((T, 5 * 64)).astype(np.float32)
    kv = mt.KV.empty(1, 2, T, {"f32": torch.float32, "f16": torch.float16, "f8": torch.uint8}[kind], gpu)
    q = torch.zeros(T, 64, device=gpu)
    mt.rope_append(torch.from_numpy(qkv).to(gpu), 1, T, 1, 2, None, kv, torch.from_numpy(INV).to(gpu), q, offset=OFFSET)
    x = qkv.reshape(T, 5, 64).astype(np.float64)
    want = np.stack([U.rope64(x[t, :3], OFFSET + t, INV) for t in range(T)])
    pair = np.abs(x[:, :3, :32]) + np.abs(x[:, :3, 32:])
    return q.cpu().numpy(), kv, want, SLACK * np.concatenate([pair, pair], -1), x[:, 3:]


def heads(t):
    return t[0].cpu().numpy().swapaxes(0, 1)  # [T, hkv, ...]


def test_queries_and_fp32_keys(gpu):
    say("fp32 keys")
    q, kv, want, slack, v = appended(gpu, "f32")
    for got, i in ((q[:, None], slice(0, 1)), (heads(kv.k), slice(1, 3))):
        assert (np.abs(got - want[:, i]) <= U.EPS32 * np.abs(want[:, i]) + slack[:, i] + 2.0 ** -149).all()
    assert np.array_equal(heads(kv.v), v)


def test_fp16_keys_are_rounded_once(gpu):
    say("fp16 keys")
    _, kv, want, slack, v = appended(gpu, "f16")
    k, s = want[:, 1:], slack[:, 1:]
    near = [(k + d * s).astype(np.float16) for d in (-1, 1)]  # the same but within the slack of a tie
    got = heads(kv.k)
    sure = near[0] == near[1]
    assert sure.mean() > 0.999 and np.array_equal(got[sure], near[0][sure])
    assert ((got == near[0]) | (got == near[1])).all()
    assert np.array_equal(heads(kv.v), v.astype(np.float16))


def test_8_bit_keys_are_the_formats_bytes(gpu):
    say("8-bit keys")
    _, kv, want, slack, v = appended(gpu, "f8")
    (ca, sa), (cb, sb) = (U.encode(want[:, 1:] + d * slack[:, 1:], 64) for d in (-1, 1))
    scales, codes = heads(kv.k_scale), heads(kv.k)
    same = sa[..., 0] == sb[..., 0]
    assert same.mean() > 0.999 and np.array_equal(scales[same], sa[..., 0][same])
    sure = (ca == cb) & same[..., None]
    assert sure.mean() > 0.999 and np.array_equal(codes[sure], ca[sure])
    assert ((codes == ca) | (codes == cb))[same].all()
    cv, sv = U.encode(v, 64)
    assert np.array_equal(heads(kv.v), cv) and np.array_equal(heads(kv.v_scale), sv[..., 0])
