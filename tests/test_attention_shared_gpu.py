"""mt_attention_shared against 64 bits, row by row: every cache type, shared prefixes and none, ragged rows, windows,
head layouts, slots past the cache, values that a row must not see."""
import numpy as np
import pytest
import torch

import mingtts as mt
import _f8_util as U
from _gpu_util import say

pytestmark = pytest.mark.gpu


class Case:
    """Inputs on the device and in 64 bits."""

    def __init__(self, gpu, kind, B, T, hq, hkv, cap, P=0, pos=None, counts=None, seed=0, q_scale=1.0):
        rng = np.random.default_rng(seed + B * 1000 + T * 10 + cap + P)
        self.B, self.T, self.hq, self.hkv, self.cap, self.P, self.kind, self.gpu = B, T, hq, hkv, cap, P, kind, gpu
        self.q = (rng.standard_normal((B * T, hq * 64)) * q_scale).astype(np.float32)
        self.own = [U.cache((B, hkv, cap), kind, rng, gpu) for _ in range(2)]
        self.pre = [U.cache((hkv, (P + 3) // 4 * 4), kind, rng, gpu) for _ in range(2)] if P else None
        self.pos = [int(rng.integers(0, cap - T + 1)) for _ in range(B)] if pos is None else pos
        self.counts = counts
        kv = lambda c: mt.KV(c[0][0], c[1][0], c[0][1], c[1][1]) if c else None  # noqa: E731
        self.kv, self.prefix = kv(self.own), kv(self.pre)

    def run(self, window=0, len_max=0, scale=0.125, stream=None, workspace=None, pad=0):
        i = lambda a: None if a is None else torch.tensor(a, dtype=torch.int32, device=self.gpu)  # noqa: E731
        q = torch.zeros(self.B * self.T, self.hq * 64 + pad, device=self.gpu)
        q[:, :self.hq * 64] = torch.from_numpy(self.q).to(self.gpu)
        out = torch.full((self.B * self.T + 1, self.hq * 64 + pad), -5.0, device=self.gpu)
        torch.cuda.synchronize()
        mt.attention_shared(q, self.B, self.T, self.hq, self.hkv, i(self.pos), self.kv, out, prefix=self.prefix, prefix_len=self.P,
                            window=window, counts=i(self.counts), len_max=len_max, scale=scale, stream=stream, workspace=workspace)
        torch.cuda.synchronize()
        out = out.cpu().double().numpy()
        assert (out[-1] == -5).all() and (out[:, self.hq * 64:] == -5).all()
        return out[:-1, :self.hq * 64].reshape(self.B, self.T, self.hq, 64)

    def want(self, b, t, h, window=0, scale=0.125):
        kh = h // (self.hq // self.hkv)
        k, v = (np.concatenate([p[2][kh, :self.P], o[2][b, kh]]) if self.P else o[2][b, kh]
                for p, o in zip(self.pre or (None, None), self.own))
        hi = self.P + min(self.pos[b] + t, self.cap - 1) + 1
        lo = max(0, hi - window) if window else 0
        return U.attend64(self.q.reshape(self.B, self.T, self.hq, 64)[b, t, h].astype(np.float64), k, v, lo, hi, scale)

    def check(self, got, window=0, scale=0.125, rows=None):
        err = norm = 0.0
        for b in range(self.B):
            for t in range(self.T):
                if t >= (self.T if self.counts is None else self.counts[b]):
                    assert (got[b, t] == -5).all()
                    continue
                if rows is not None and (b, t) not in rows:
                    continue
                for h in range(self.hq):
                    want, tol = self.want(b, t, h, window, scale)
                    worst = np.abs(got[b, t, h] - want).max()
                    assert worst <= tol, f"row {b} {t} head {h}: off by {worst:.3g}, bound {tol:.3g}"
                    err += ((got[b, t, h] - want) ** 2).sum()
                    norm += (want ** 2).sum()
        rel = np.sqrt(err / norm)
        assert rel <= 5e-6, rel
        return rel


SHAPES = [
    # B, T, hq, hkv, cap, P
    (1, 1, 1, 1, 4, 0),
    (2, 1, 14, 2, 512, 0),
    (2, 1, 14, 2, 512, 174),
    (1, 1, 14, 2, 40, 1),
    (5, 1, 16, 16, 132, 33),
    (3, 1, 16, 1, 260, 95),
    (40, 1, 8, 2, 64, 200),
    (2, 1, 40, 2, 72, 31),
    (1, 1, 14, 2, 5000, 0),
    (1, 1, 4, 4, 36, 3000),
    (2, 9, 14, 2, 64, 0),
    (3, 17, 12, 4, 48, 70),
    (2, 50, 14, 2, 100, 33),
    (1, 130, 4, 1, 200, 129),
]


@pytest.mark.parametrize("kind", ["f32", "f16", "f8"])
@pytest.mark.parametrize("shape", SHAPES)
def test_attention(gpu, kind, shape):
    say(f"attention {kind} {shape}")
    B, T, hq, hkv, cap, P = shape
    c = Case(gpu, kind, *shape)
    c.check(c.run(pad=4))


@pytest.mark.parametrize("kind", ["f32", "f16", "f8"])
@pytest.mark.parametrize("B,T,pos,counts", [
    (4, 1, [0, 0, 63, 62], None),
    (4, 1, [0, 31, 32, 33], [1, 0, 1, 1]),
    (3, 6, [0, 58, 20], [1, 6, 0]),
    (3, 6, [60, 64, 1000], [6, 2, 1]),  # rows past the cache attend all of it
    (2, 40, [0, 24], [33, 40]),
])
@pytest.mark.parametrize("P", [0, 45])
def test_ragged(gpu, kind, B, T, pos, counts, P):
    say(f"ragged {kind} {B} {T} {P}")
    c = Case(gpu, kind, B, T, 14, 2, 64, P, pos=pos, counts=counts)
    c.check(c.run())


@pytest.mark.parametrize("kind", ["f32", "f16", "f8"])
@pytest.mark.parametrize("window", [1, 5, 64, 65, 200, 10000])
@pytest.mark.parametrize("B,T,cap,P", [(3, 1, 128, 100), (2, 20, 64, 77), (70, 1, 64, 150)])
def test_window(gpu, kind, window, B, T, cap, P):
    say(f"window {kind} {window} {B} {T}")
    c = Case(gpu, kind, B, T, 14, 2, cap, P)
    c.check(c.run(window=window), window=window)


@pytest.mark.parametrize("kind", ["f32", "f16", "f8"])
def test_long_split_and_hints(gpu, kind):
    """Few rows over many keys, and bounds of the length that are too small, exact and too large."""
    c = Case(gpu, kind, 2, 1, 14, 2, 20000, 0, pos=[19999, 12345])
    for len_max in (0, 1, 700, 20000):
        c.check(c.run(len_max=len_max))
    c = Case(gpu, kind, 2, 2, 8, 2, 9000, 6001, pos=[8998, 17], counts=[2, 1])
    for len_max in (0, 40, 9000):
        c.check(c.run(len_max=len_max))


@pytest.mark.parametrize("kind", ["f32", "f16", "f8"])
@pytest.mark.parametrize("scale,q_scale", [(0.125, 30.0), (-0.2, 3.0), (1.0, 1e-3), (1e-6, 1.0), (0.0, 1.0)])
def test_scales_of_the_scores(gpu, kind, scale, q_scale):
    c = Case(gpu, kind, 3, 2, 14, 2, 96, 50, q_scale=q_scale)
    c.check(c.run(scale=scale), scale=scale)


def test_blocks_of_very_different_sizes(gpu):
    """8-bit values whose scales lie 2^30 apart from key to key."""
    c = Case(gpu, "f8", 2, 3, 14, 2, 64, 40)
    rng = np.random.default_rng(1)
    for group in (c.own, c.pre):
        for i, (codes, scales, _) in enumerate(group):
            s = scales.cpu().numpy().astype(int) + (rng.integers(-30, 31, scales.shape) if i else rng.integers(-4, 2, scales.shape))
            scales.copy_(torch.from_numpy(s.astype(np.uint8)))
            group[i] = (codes, scales, U.decode(codes.cpu().numpy(), s[..., None], 64))
    c.check(c.run())


@pytest.mark.parametrize("kind", ["f32", "f16", "f8"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf"), 6e4])
@pytest.mark.parametrize("P,window", [(0, 0), (70, 0), (70, 30)])
def test_what_a_row_does_not_attend(gpu, kind, bad, P, window):
    """Slots behind a row's own (later rows' keys and stale ones), padding of the prefix, keys before the window, other
    sequences and padding rows' queries hold values that must not reach it."""
    say(f"unattended {kind} {bad} {P} {window}")
    B, T, cap = 3, 6, 96
    c = Case(gpu, kind, B, T, 14, 2, cap, P, pos=[20, 31, 0], counts=[6, 3, 1])
    clean = c.run(window=window)
    c.check(clean, window=window)
    later = (1, 2)  # sequence 1's last row: its key reaches that row alone
    for codes, scales, _ in c.own:
        for b in range(B):
            at = slice(c.pos[b] + c.counts[b] - (b == 1), cap)
            if scales is None:
                codes[b, :, at] = bad
            elif bad == bad and abs(bad) < 1e9:
                scales[b, :, at] = 247
            else:
                codes[b, :, at] = 127
    if P:
        for codes, scales, _ in c.pre:
            codes[:, P:] = 127 if kind == "f8" else bad
            if window and kind != "f8":
                codes[:, :P - window] = bad  # every row's window starts behind these
            elif window:
                codes[:, :P - window] = 127
    for b in range(B):
        c.q.reshape(B, T, 14, 64)[b, c.counts[b]:] = bad
    dirty = c.run(window=window)
    for b in range(B):
        for t in range(T):
            if (b, t) != later and t < c.counts[b]:
                # the same keys and weights: what the rounding order may change is bounded as in check()
                for h in range(14):
                    want, tol = c.want(b, t, h, window)
                    assert np.abs(dirty[b, t, h] - want).max() <= tol, (b, t, h)


def test_scores_that_are_not_finite(gpu):
    """As the formula has it: a NaN or +infinity among a row's scores makes it NaN, a -infinity is no weight,
    nothing but -infinity is NaN; other rows keep their results."""
    c = Case(gpu, "f32", 2, 4, 2, 2, 64, 0, pos=[10, 40])
    clean = c.run()
    k = c.own[0][0]
    q = c.q.reshape(2, 4, 2, 64)
    q[:, :, :, 0] = 1.0
    base = c.run()
    k[0, 0, 3, 0], k[0, 1, 5, 0] = float("nan"), float("inf")
    k[1, 0, 7, 0] = -float("inf")
    k[1, 1, :, 0] = -float("inf")
    got = c.run()
    assert np.isnan(got[0]).all() and np.isnan(got[1, :, 1]).all()
    x = c.own[0][2].copy()
    x[1, 0, 7, 0] = -1e30
    for t in range(4):
        want, tol = U.attend64(q[1, t, 0].astype(np.float64), x[1, 0], c.own[1][2][1, 0], 0, 41 + t, 0.125)
        # the key of -1e30 has no weight and no part in the other scores' error
        assert np.abs(got[1, t, 0] - want).max() <= 1e-4
    assert np.isfinite(clean).all() and np.isfinite(base).all()


def test_prefix_is_one_cache_for_all(gpu):
    """The shared prefix gives what each sequence gets with the prefix copied into its own cache."""
    c = Case(gpu, "f8", 6, 2, 14, 2, 64, 40)
    got = c.run()
    own = [torch.cat([p[0][None].expand(6, -1, -1, -1)[:, :, :40], o[0]], 2).contiguous() for p, o in zip(c.pre, c.own)]
    sc = [torch.cat([p[1][None].expand(6, -1, -1)[:, :, :40], o[1]], 2).contiguous() for p, o in zip(c.pre, c.own)]
    d = Case(gpu, "f8", 6, 2, 14, 2, 104, 0, pos=[p + 40 for p in c.pos])
    d.q, d.kv = c.q, mt.KV(own[0], own[1], sc[0], sc[1])
    d.own = [(o, s, U.decode(o.cpu().numpy(), s.cpu().numpy()[..., None], 64)) for o, s in zip(own, sc)]
    alone = d.run()
    c.check(got)
    d.check(alone)


def test_a_strided_batch(gpu):
    c = Case(gpu, "f8", 3, 1, 14, 2, 64, 0)
    wide = []
    for codes, scales, _ in c.own:
        a = torch.full((6, 2, 64, 64), 127, dtype=torch.uint8, device=gpu)
        s = torch.full((6, 2, 64), 5, dtype=torch.uint8, device=gpu)
        a[::2], s[::2] = codes, scales
        wide.append((a, s))
    want = c.run()
    c.kv = mt.KV(wide[0][0][::2], wide[1][0][::2], wide[0][1][::2], wide[1][1][::2])
    assert np.array_equal(c.run(), want)


def test_a_cache_past_32_bit_offsets(gpu):
    """An fp16 cache of 2^25 + 64 slots: the second head starts past 2^32 bytes, and so do the keys of a window at its end."""
    cap = (1 << 25) + 64
    k = torch.zeros(2, cap, 64, dtype=torch.float16, device=gpu)
    v = torch.zeros_like(k)
    rng = np.random.default_rng(2)
    n = 200
    kx, vx = (rng.standard_normal((2, n, 64)).astype(np.float16) for _ in range(2))
    k[:, cap - n:], v[:, cap - n:] = torch.from_numpy(kx).to(gpu), torch.from_numpy(vx).to(gpu)
    q = rng.standard_normal((1, 256)).astype(np.float32)
    out = torch.zeros(1, 256, device=gpu)
    mt.attention_shared(torch.from_numpy(q).to(gpu), 1, 1, 4, 2, torch.tensor([cap - 1], dtype=torch.int32, device=gpu), mt.KV(k, v), out,
                        window=150)
    for h in range(4):
        want, tol = U.attend64(q.reshape(4, 64)[h].astype(np.float64), kx[h // 2].astype(np.float64), vx[h // 2].astype(np.float64), n - 150, n,
                               0.125)
        assert np.abs(out.cpu().numpy().reshape(4, 64)[h] - want).max() <= tol


@pytest.mark.parametrize("shape", [(2, 1, 14, 2, 512, 0), (1, 1, 14, 2, 9000, 0), (70, 1, 14, 2, 64, 600), (3, 20, 14, 2, 64, 50)])
def test_graph_replays_and_streams(gpu, shape):
    """Replays with other lengths give the eager result; two graphs at once on two streams, each with the workspace
    of its capture, too; a call gives the same bits every time."""
    c = Case(gpu, "f8", *shape)
    B, T, hq, hkv, cap, P = shape
    q = torch.from_numpy(c.q).to(gpu)
    pos = torch.tensor(c.pos, dtype=torch.int32, device=gpu)

    def call(out, p, stream=None):
        mt.attention_shared(q, B, T, hq, hkv, p, c.kv, out, prefix=c.prefix, prefix_len=P, stream=stream)

    outs, poss, graphs = [], [], []
    for i in range(2):
        out, p = torch.zeros(B * T, hq * 64, device=gpu), pos.clone()
        call(out, p)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call(out, p)
        outs.append(out), poss.append(p), graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(2)]
    want = [torch.zeros_like(outs[0]) for _ in range(2)]
    for r in range(4):
        for i in range(2):
            poss[i].copy_(torch.clamp(pos - r * (i + 1), min=0))
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            call(want[i], poss[i])
            assert torch.equal(want[i], outs[i]), (r, i)
    # explicit streams, workspaces from the allocator
    a, b = torch.zeros_like(want[0]), torch.zeros_like(want[0])
    torch.cuda.synchronize()
    call(a, poss[0], streams[0])
    call(b, poss[1], streams[1])
    torch.cuda.synchronize()
    assert torch.equal(a, want[0]) and torch.equal(b, want[1])


@pytest.mark.parametrize("byte", [0, 255])
@pytest.mark.parametrize("P,window", [(0, 0), (70, 0), (6001, 0)])
def test_stale_scale_bytes(gpu, byte, P, window):
    """Scale bytes of slots that no row attends, behind a sequence's end and the prefix's, are not values: any byte may
    stand there, in one pass and in parts."""
    c = Case(gpu, "f8", 2, 2, 14, 2, 64, P, pos=[20, 45], counts=[2, 1])
    want = c.run(window=window)
    for _, scales, _ in c.own:
        scales[0, :, 22:], scales[1, :, 46:] = byte, byte
    for _, scales, _ in c.pre or ():
        scales[:, P:] = byte
    assert np.array_equal(c.run(window=window), want)
