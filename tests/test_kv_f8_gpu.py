"""mt_rope_append and mt_kv_copy against 64 bits: every cache type, ragged rows, slots past the cache, far positions,
special values, guard bytes around everything that must stay as it was."""
import numpy as np
import pytest
import torch

import mingtts as mt
import _f8_util as U
from _gpu_util import say

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "f16": torch.float16, "f8": torch.uint8}
INV = (1.0 / 1e6 ** (np.arange(32) / 32)).astype(np.float32)


def values(kv, name):
    """A cache's values in 64 bits."""
    x = getattr(kv, name).cpu()
    if kv.type != mt.F8:
        return x.double().numpy()
    return U.decode(x.view(torch.uint8).numpy(), getattr(kv, name + "_scale").cpu().numpy()[..., None], 64)


def run_append(gpu, kind, B, T, hq, hkv, cap, pos, counts, offset, qkv, q=True, pad=0):
    """The call on guarded buffers; returns the caches, q (or None) and the host's inputs."""
    width = (hq + 2 * hkv) * 64
    buf = torch.full((B * T, width + pad), 7.0, device=gpu)
    buf[:, :width] = torch.from_numpy(qkv).to(gpu)
    kv = mt.KV.empty(B, hkv, cap, TYPES[kind], gpu)
    for t in (kv.k, kv.v):
        t.fill_(3)
    out = torch.full((B * T + 1, hq * 64 + pad), -5.0, device=gpu) if q else None
    d = lambda a: None if a is None else torch.tensor(a, dtype=torch.int32, device=gpu)  # noqa: E731
    mt.rope_append(buf, B, T, hq, hkv, d(pos), kv, torch.from_numpy(INV).to(gpu), out, counts=d(counts), offset=offset)
    torch.cuda.synchronize()
    bits = buf[:, :width].contiguous().view(torch.int32).cpu()  # NaN too
    assert torch.equal(bits, torch.from_numpy(qkv.view(np.int32))) and bool((buf[:, width:] == 7).all())
    return kv, out


def check_append(kv, out, kind, B, T, hq, hkv, cap, pos, counts, offset, qkv):
    x = qkv.reshape(B, T, hq + 2 * hkv, 64).astype(np.float64)
    untouched = np.ones((B, hkv, cap), bool)
    for b in range(B):
        for t in range(T):
            have, slot = t < (T if counts is None else counts[b]), (0 if pos is None else pos[b]) + t
            if out is not None:
                got = out[b * T + t, :hq * 64].cpu().double().numpy().reshape(hq, 64)
                if not have:
                    assert (got == -5).all()
                else:
                    want = U.rope64(x[b, t, :hq], offset + slot, INV)
                    # The turn's rounding (9.4e-8 rad), sine and cosine within 2 ulp, three roundings of the rotation: 4e-7
                    # of |x0| + |x1|.
                    pair = np.abs(x[b, t, :hq, :32]) + np.abs(x[b, t, :hq, 32:])
                    assert (np.abs(got - want) <= 5e-7 * np.concatenate([pair, pair], -1)).all()
            if not have or slot >= cap:
                continue
            untouched[b, :, slot] = False
            want = {"k": U.rope64(x[b, t, hq:hq + hkv], offset + slot, INV), "v": x[b, t, hq + hkv:]}
            pair = np.abs(x[b, t, hq:hq + hkv, :32]) + np.abs(x[b, t, hq:hq + hkv, 32:])
            slack = {"k": 5e-7 * np.concatenate([pair, pair], -1), "v": 0.0}
            for n in ("k", "v"):
                got = values(kv, n)[b, :, slot]
                if kind == "f8":
                    s = 2.0 ** (getattr(kv, n + "_scale")[b, :, slot].cpu().numpy().astype(float) - 127)
                    half = np.maximum(np.abs(want[n]) * 2.0 ** -4, 2.0 ** -10 * s[:, None])
                else:
                    half = np.abs(want[n]) * (2.0 ** -11 if kind == "f16" else U.EPS32) + 2.0 ** -25
                assert (np.abs(got - want[n]) <= half + slack[n] * 1.001).all(), (n, b, t)
                if kind == "f8" and n == "v":  # no arithmetic before the rounding: the format's own bytes
                    c, sb = U.encode(want[n], 64)
                    assert np.array_equal(kv.v[b, :, slot].cpu().numpy(), c) and np.array_equal(kv.v_scale[b, :, slot].cpu().numpy(), sb[:, 0])
    for n in ("k", "v"):
        raw = getattr(kv, n).cpu().float().numpy()
        assert (raw[untouched] == 3).all()
        if kind == "f8":
            assert (getattr(kv, n + "_scale").cpu().numpy()[untouched] == 1).all()


CASES = [
    # B, T, hq, hkv, cap, pos, counts, offset
    (2, 1, 14, 2, 512, [5, 511], None, 0),
    (1, 1, 1, 1, 4, [0], None, 0),
    (1, 1, 14, 2, 16, None, None, 0),
    (3, 5, 14, 2, 32, [0, 30, 40], [5, 4, 2], 174),  # rows past the cache append nothing
    (4, 7, 16, 16, 12, [0, 1, 2, 3], [0, 7, 1, 3], 0),
    (2, 300, 12, 4, 304, [0, 3], [300, 257], 9),      # more than 512 rows: four to a workgroup
    (5, 3, 8, 1, 8, [1, 2, 3, 4, 5], None, 131072),
]


@pytest.mark.parametrize("kind", ["f32", "f16", "f8"])
@pytest.mark.parametrize("case", CASES)
def test_append(gpu, kind, case):
    B, T, hq, hkv, cap, pos, counts, offset = case
    say(f"append {kind} {case[:5]}")
    rng = np.random.default_rng(B * 100 + T)
    qkv = rng.standard_normal((B * T, (hq + 2 * hkv) * 64)).astype(np.float32)
    kv, out = run_append(gpu, kind, B, T, hq, hkv, cap, pos, counts, offset, qkv, pad=4 * (T % 3))
    check_append(kv, out, kind, *case, qkv)
    assert bool((out[-1] == -5).all()) and bool((out[:, hq * 64:] == -5).all())


def test_append_without_q_and_in_place(gpu):
    rng = np.random.default_rng(3)
    qkv = rng.standard_normal((6, 18 * 64)).astype(np.float32)
    case = (3, 2, 14, 2, 32, [4, 5, 6], None, 11)
    kv, _ = run_append(gpu, "f8", *case, qkv, q=False)
    check_append(kv, None, "f8", *case, qkv)
    kv2, out = run_append(gpu, "f8", *case, qkv)
    buf = torch.from_numpy(qkv).to(gpu)
    kv3 = mt.KV.empty(3, 2, 32, torch.uint8, gpu)
    mt.rope_append(buf, 3, 2, 14, 2, torch.tensor([4, 5, 6], dtype=torch.int32, device=gpu), kv3, torch.from_numpy(INV).to(gpu), buf, offset=11)
    assert torch.equal(buf[:, :896], out[:-1, :896]) and torch.equal(buf[:, 896:].cpu(), torch.from_numpy(qkv[:, 896:]))
    at = (slice(None), slice(None), slice(4, 6))
    assert torch.equal(kv3.k[at][0], kv2.k[at][0]) and torch.equal(kv3.k_scale[at][0], kv2.k_scale[at][0])


def test_append_special_values(gpu):
    """Zeros, subnormals, the largest values, infinities and NaN, and blocks at the edges of a scale."""
    rows = np.zeros((8, 3 * 64), np.float32)
    v = rows[:, 128:]
    v[1] = 2.0 ** -140
    v[2, :3] = [3.4e38, -3.0e38, 1.0]
    v[3, :5] = [1.0, np.inf, -np.inf, np.nan, 0.3]
    v[4, :2] = [448.0, 1e-3]
    v[5, :2] = [np.nextafter(np.float32(448), np.float32(449)), 1.0]
    v[6] = np.nan
    v[7] = np.linspace(-1, 1, 64)
    kv, _ = run_append(gpu, "f8", 8, 1, 1, 1, 4, [0] * 8, None, 0, rows)
    c, s = U.encode(v.astype(np.float64), 64)
    got, gs = kv.v[:, 0, 0].cpu().numpy(), kv.v_scale[:, 0, 0].cpu().numpy()
    nan = (c & 127) == 127
    assert np.array_equal(gs, s[:, 0])
    assert np.array_equal(got[~nan], c[~nan]) and ((got[nan] & 127) == 127).all()


@pytest.mark.parametrize("src", ["f32", "f16", "f8"])
@pytest.mark.parametrize("dst", ["f32", "f16", "f8"])
def test_copy(gpu, src, dst):
    rng = np.random.default_rng(7)
    B, hkv, pos, counts, T = 3, 2, [0, 5, 14], [6, 0, 6], 6
    parts = [U.cache((B, hkv, 20), src, rng, gpu) for _ in range(2)]
    s = mt.KV(parts[0][0], parts[1][0], parts[0][1], parts[1][1])
    d = mt.KV.empty(B, hkv, 16, TYPES[dst], gpu)  # a shorter cache: slots past it are left out
    for t in (d.k, d.v):
        t.fill_(3)
    i = lambda a: torch.tensor(a, dtype=torch.int32, device=gpu)  # noqa: E731
    mt.kv_copy(s, d, B, T, pos=i(pos), counts=i(counts))
    torch.cuda.synchronize()
    left = np.ones((B, hkv, 16), bool)
    for n, (_, _, x) in zip(("k", "v"), parts):
        got = values(d, n)
        for b in range(B):
            for t in range(counts[b]):
                at = pos[b] + t
                if at >= 16:
                    continue
                left[b, :, at] = False
                want = x[b, :, at]
                if dst == "f8":
                    want = U.decode(*U.encode(want, 64), 64)
                elif dst == "f16":
                    want = want.astype(np.float16).astype(np.float64)
                assert np.array_equal(got[b, :, at], want)
        assert (getattr(d, n).cpu().float().numpy()[left] == 3).all()


def test_a_strided_batch_and_the_whole_prompt(gpu):
    """Caches that are every second sequence of a larger tensor; a copy without pos takes slots 0 .. T - 1."""
    rng = np.random.default_rng(8)
    big = [U.cache((4, 2, 40), "f8", rng, gpu) for _ in range(2)]
    s = mt.KV(big[0][0][::2], big[1][0][::2], big[0][1][::2], big[1][1][::2])
    d = mt.KV.empty(2, 2, 40, torch.float32, gpu)
    mt.kv_copy(s, d, 2, 40)
    assert np.array_equal(values(d, "k"), big[0][2][::2]) and np.array_equal(values(d, "v"), big[1][2][::2])
    back = mt.KV.empty(2, 2, 40, torch.uint8, gpu)
    mt.kv_copy(d, back, 2, 40)  # the values again, whatever scale their bytes take
    assert np.array_equal(values(back, "k"), big[0][2][::2])


def test_a_cache_past_32_bit_offsets(gpu):
    """Slots whose byte offset passes 2^32: an fp32 cache of 2^24 + 64 slots and two heads."""
    cap = (1 << 24) + 64
    k = torch.empty(2, cap, 64, device=gpu)
    kv = mt.KV(k, torch.empty_like(k))
    pos = cap - 3
    rng = np.random.default_rng(9)
    qkv = rng.standard_normal((3, 6 * 64)).astype(np.float32)
    mt.rope_append(torch.from_numpy(qkv).to(gpu), 1, 3, 2, 2, torch.tensor([pos], dtype=torch.int32, device=gpu), kv,
                   torch.from_numpy(INV).to(gpu))
    got = kv.v[:, pos:].cpu().numpy()
    assert np.array_equal(got, qkv.reshape(3, 6, 64)[:, 4:].transpose(1, 0, 2))
    want = np.stack([U.rope64(qkv.reshape(3, 6, 64)[t, 2:4].astype(np.float64), pos + t, INV) for t in range(3)], 1)
    assert np.abs(kv.k[:, pos:].cpu().numpy() - want).max() <= 5e-7 * 2 * np.abs(qkv).max()


def test_graph_replays(gpu):
    rng = np.random.default_rng(10)
    qkv = torch.from_numpy(rng.standard_normal((4, 18 * 64)).astype(np.float32)).to(gpu)
    pos = torch.zeros(4, dtype=torch.int32, device=gpu)
    inv = torch.from_numpy(INV).to(gpu)
    kv, q = mt.KV.empty(4, 2, 64, torch.uint8, gpu), torch.zeros(4, 896, device=gpu)
    f = mt.KV.empty(4, 2, 64, torch.float32, gpu)

    def step(c, o, r):
        mt.rope_append(qkv, 4, 1, 14, 2, pos, c, inv, o)
        mt.kv_copy(c, r, 4, 1, pos=pos)

    step(kv, q, f)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(kv, q, f)
    kv2, q2, f2 = mt.KV.empty(4, 2, 64, torch.uint8, gpu), torch.zeros(4, 896, device=gpu), mt.KV.empty(4, 2, 64, torch.float32, gpu)
    step(kv2, q2, f2)
    for i in range(4):
        pos.add_(3)
        qkv.mul_(1.25)
        graph.replay()
        step(kv2, q2, f2)
        torch.cuda.synchronize()
        for a, b in ((kv.k, kv2.k), (kv.v_scale, kv2.v_scale), (q, q2), (f.k, f2.k), (f.v, f2.v)):
            assert torch.equal(a, b), i
