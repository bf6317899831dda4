"""8-bit blocks of all scales read back: what comes out is what the bytes stand for, the smallest blocks among them."""
import numpy as np
import pytest
import torch

import mingtts as mt
import _f8_util as U
from _gpu_util import say
from test_attention_shared_gpu import Case

pytestmark = pytest.mark.gpu
SCALES = [1, 2, 3, 4, 9, 100, 127, 150, 246, 247, 254]


def all_codes(gpu, dtype):
    """Every code under the least, middle and largest scale bytes, copied into another type."""
    n = 4 * len(SCALES)
    codes = np.tile(np.arange(256, dtype=np.uint8).reshape(4, 64), (len(SCALES), 1)).reshape(1, 1, n, 64)
    scales = np.repeat(np.array(SCALES, np.uint8), 4).reshape(1, 1, n)
    c, s = torch.from_numpy(codes).to(gpu), torch.from_numpy(scales).to(gpu)
    src = mt.KV(c, c.clone(), s, s.clone())
    dst = mt.KV.empty(1, 1, n, dtype, gpu)
    mt.kv_copy(src, dst, 1, n)
    return U.decode(codes, scales[..., None], 64), dst


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_every_code_reads_back_exactly(gpu, dtype):
    """Into fp32 as it is (past fp32's range: infinity); into fp16 with that type's one rounding."""
    say(f"read back {dtype}")
    want, dst = all_codes(gpu, dtype)
    with np.errstate(over="ignore"):
        want = want.astype(np.float32 if dtype == torch.float32 else np.float16)
    for t in (dst.k, dst.v):
        assert np.array_equal(t.cpu().numpy(), want, equal_nan=True)


@pytest.mark.parametrize("M", [3, 70])
def test_the_smallest_blocks_in_a_product(gpu, M):
    """Blocks under scale bytes 1 to 4 as weights: the matrix cores take them as bf16, a step of 2^-133 at the least."""
    say(f"smallest blocks {M}")
    rng = np.random.default_rng(3)
    N, K = 33, 512
    codes = rng.integers(0, 256, (N, K)).astype(np.uint8)
    codes[(codes & 127) == 127] = 1
    codes[:11] &= 0x87  # the smallest steps alone
    scales = np.tile(np.array([1, 2, 3, 4], np.uint8), (N, 1))
    w = mt.F8Matrix(torch.from_numpy(codes).to(gpu), torch.from_numpy(scales).to(gpu))
    x = mt.F8Matrix.quantize(torch.from_numpy((rng.standard_normal((M, K)) * 2.0 ** 100).astype(np.float32)).to(gpu))
    y = torch.zeros(M, N, device=gpu)
    mt.linear_f8(x, w, y)
    x64, w64 = U.decode(x.codes.cpu().numpy(), x.scales.cpu().numpy(), 128), U.decode(codes, scales, 128)
    # half a bf16 step of each weight beside the sums' whole fp32 steps
    tol = np.abs(x64).sum(1)[:, None] * 2.0 ** -134 + (K / 16 + 64) * 2 * U.EPS32 * (np.abs(x64) @ np.abs(w64).T)
    assert (np.abs(y.cpu().numpy() - x64 @ w64.T) <= tol).all()


@pytest.mark.parametrize("P", [0, 8192])
def test_the_smallest_blocks_in_attention(gpu, P):
    """Keys and values under scale bytes 1 to 20, in one pass and in parts."""
    say(f"smallest blocks, attention {P}")
    c = Case(gpu, "f8", 3, 1, 14, 2, 512, P)
    rng = np.random.default_rng(4)
    for group in filter(None, (c.own, c.pre)):
        for i, (codes, scales, _) in enumerate(group):
            s = rng.integers(1, 21, tuple(scales.shape)).astype(np.uint8)
            scales.copy_(torch.from_numpy(s))
            group[i] = (codes, scales, U.decode(codes.cpu().numpy(), s[..., None], 64))
    got = c.run(scale=2.0 ** 100)
    for b in range(3):
        for h in range(14):
            want, tol = c.want(b, 0, h, 0, 2.0 ** 100)
            assert np.abs(got[b, 0, h] - want).max() <= tol + (P + c.pos[b] + 1) * 2.0 ** -125
