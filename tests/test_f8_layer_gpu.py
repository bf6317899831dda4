"""The 8-bit operators together, as a serving loop uses them: a voice prompt prefilled once and set aside as an 8-bit
prefix, ragged texts behind it, decode steps of the batch.  Every call is checked in 64 bits on the inputs it was
given (the outputs of the call before), eagerly and as one captured graph."""
import numpy as np
import pytest
import torch

import mingtts as mt
import _f8_util as U
from _gpu_util import say

pytestmark = pytest.mark.gpu
F = mt.GemvFlags
H, HQ, HKV, MLP, CAP = 256, 4, 2, 528, 64
INV = (1.0 / 1e4 ** (np.arange(32) / 32)).astype(np.float32)


class Layer:
    def __init__(self, gpu, seed=0):
        rng = np.random.default_rng(seed)
        self.gpu, self.w = gpu, {}
        for name, n, k in (("qkv", (HQ + 2 * HKV) * 64, H), ("o", H, HQ * 64), ("gate", MLP, H), ("up", MLP, H), ("down", H, MLP)):
            self.w[name] = mt.F8Matrix.quantize(torch.from_numpy(rng.standard_normal((n, k)).astype(np.float32) * 0.08).to(gpu))
        self.bias = torch.from_numpy(rng.standard_normal((HQ + 2 * HKV) * 64) * 0.1).to(torch.float16).to(gpu)
        self.norms = [torch.from_numpy(1 + 0.1 * rng.standard_normal(H)).to(torch.float16).to(gpu) for _ in range(2)]
        self.inv = torch.from_numpy(INV).to(gpu)

    def buffers(self, rows):
        z = lambda n: torch.zeros(rows, n, device=self.gpu)  # noqa: E731
        return dict(qkv=z((HQ + 2 * HKV) * 64), q=z(HQ * 64), att=z(HQ * 64), mlp=z(MLP))

    def step(self, x, b, B, T, pos, kv, prefix, P, counts=None, seen=None):
        """x (fp32 [B T, H], updated in place) through the layer; `seen` gets each call's inputs and outputs."""
        note = lambda n, v: seen.__setitem__(n, v.clone()) if seen is not None else None  # noqa: E731
        note("x0", x)
        mt.linear_f8(x, self.w["qkv"], b["qkv"], bias=self.bias, norm=self.norms[0])
        mt.rope_append(b["qkv"], B, T, HQ, HKV, pos, kv, self.inv, b["q"], counts=counts, offset=P)
        mt.attention_shared(b["q"], B, T, HQ, HKV, pos, kv, b["att"], prefix=prefix, prefix_len=P, counts=counts)
        mt.linear_f8(b["att"], self.w["o"], x, flags=F.accumulate)
        note("x1", x)
        mt.linear_f8(x, self.w["gate"], b["mlp"], flags=F.siluGate, w2=self.w["up"], norm=self.norms[1])
        mt.linear_f8(b["mlp"], self.w["down"], x, flags=F.accumulate)
        note("x2", x)


def dec(m):
    return U.decode(m.codes.cpu().numpy(), m.scales.cpu().numpy(), 128)


def check_linear(x, w, got, old=None, norm=None, w2=None, bias=None, what=""):
    """got = old + epilogue(quantised x . w): x64 is the quantiser's own bytes (its tests hold those), products exact,
    sums of K / 16 + 64 whole fp32 steps."""
    xq = dec(mt.F8Matrix.quantize(x, norm=norm))
    r = (xq.shape[1] / 16 + 64) * 2 * U.EPS32
    y, tol = xq @ dec(w).T, r * (np.abs(xq) @ np.abs(dec(w)).T)
    if bias is not None:
        y = y + bias.double().cpu().numpy()
    if w2 is not None:
        u = xq @ dec(w2).T
        tol = 1.1 * tol * np.abs(u) + np.abs(y) * r * (np.abs(xq) @ np.abs(dec(w2)).T)
        y = y / (1 + np.exp(-y)) * u
    old = 0.0 if old is None else old.double().cpu().numpy()
    err = np.abs(got.double().cpu().numpy() - (y + old))
    assert (err <= tol + 16 * U.EPS32 * (np.abs(y) + np.abs(old) + 1)).all(), what


def values(kv, n):
    x = getattr(kv, n).cpu()
    return x.double().numpy() if kv.type != mt.F8 else U.decode(x.numpy(), getattr(kv, n + "_scale").cpu().numpy()[..., None], 64)


def check_step(layer, b, seen, B, T, pos, kv, prefix, P, counts, what):
    say(what)
    n = [T] * B if counts is None else counts
    check_linear(seen["x0"], layer.w["qkv"], b["qkv"], norm=layer.norms[0], bias=layer.bias, what=what + " qkv")
    heads = b["qkv"].double().cpu().numpy().reshape(B, T, HQ + 2 * HKV, 64)
    q, att = (b[k].double().cpu().numpy().reshape(B, T, HQ, 64) for k in ("q", "att"))
    k, v = values(kv, "k"), values(kv, "v")
    pk, pv = (values(prefix, "k"), values(prefix, "v")) if P else (None, None)
    for s in range(B):
        for t in range(n[s]):
            at = pos[s] + t
            want = U.rope64(heads[s, t, :HQ + HKV], P + at, INV)
            assert np.abs(q[s, t] - want[:HQ]).max() <= 5e-7 * 2 * np.abs(heads[s, t]).max(), what
            for got, row in ((k[s, :, at], want[HQ:]), (v[s, :, at], heads[s, t, HQ + HKV:])):
                assert np.array_equal(got, U.decode(*U.encode(row, 64), 64)), what  # the cached values are the format's own
            for h in range(HQ):
                kh = h // (HQ // HKV)
                kk, vv = (np.concatenate([p[kh, :P], o[s, kh]]) if P else o[s, kh] for p, o in ((pk, k), (pv, v)))
                want_o, tol = U.attend64(q[s, t, h], kk, vv, 0, P + at + 1, 0.125)
                assert np.abs(att[s, t, h] - want_o).max() <= tol, what
    check_linear(b["att"], layer.w["o"], seen["x1"], old=seen["x0"], what=what + " o")
    check_linear(seen["x1"], layer.w["gate"], b["mlp"], norm=layer.norms[1], w2=layer.w["up"], what=what + " gate|up")
    check_linear(b["mlp"], layer.w["down"], seen["x2"], old=seen["x1"], what=what + " down")


def test_a_prompt_shared_by_a_batch(gpu):
    layer, rng = Layer(gpu), np.random.default_rng(1)
    rand = lambda *s: torch.from_numpy(rng.standard_normal(s).astype(np.float32)).to(gpu)  # noqa: E731
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=gpu)  # noqa: E731
    # The voice prompt, prefilled alone in an 8-bit cache (37 rows: the GEMMs and a row tile's causal edge).
    P = 37
    first = mt.KV.empty(1, HKV, CAP, torch.uint8, gpu)
    x, b, seen = rand(P, H), layer.buffers(P), {}
    layer.step(x, b, 1, P, None, first, None, 0, seen=seen)
    check_step(layer, b, seen, 1, P, [0], first, None, 0, None, "voice prompt")
    # Set aside as the shared prefix, with room to spare behind it.
    prefix = mt.KV.empty(1, HKV, 40, torch.uint8, gpu)
    mt.kv_copy(first, prefix, 1, P)
    prefix = mt.KV(prefix.k[0], prefix.v[0], prefix.k_scale[0], prefix.v_scale[0])
    assert torch.equal(prefix.k[:, :P], first.k[0, :, :P]) and torch.equal(prefix.v_scale[:, :P], first.v_scale[0, :, :P])
    # Three texts of different lengths behind it.
    B, T, counts = 3, 9, [9, 4, 6]
    kv = mt.KV.empty(B, HKV, CAP, torch.uint8, gpu)
    x, b, seen = rand(B * T, H), layer.buffers(B * T), {}
    layer.step(x, b, B, T, None, kv, prefix, P, counts=i32(counts), seen=seen)
    check_step(layer, b, seen, B, T, [0] * B, kv, prefix, P, counts, "texts")
    # Decode steps, captured once: every replay against the eager step on a copy of the caches and against 64 bits.
    x, b, pos = torch.zeros(B, H, device=gpu), layer.buffers(B), i32(counts)
    twin = mt.KV(kv.k.clone(), kv.v.clone(), kv.k_scale.clone(), kv.v_scale.clone())
    keep = [t.clone() for t in (kv.k, kv.v, kv.k_scale, kv.v_scale)]
    layer.step(x, b, B, 1, pos, kv, prefix, P)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer.step(x, b, B, 1, pos, kv, prefix, P)
    for t, k in zip((kv.k, kv.v, kv.k_scale, kv.v_scale), keep):
        t.copy_(k)
    for n in range(4):
        inp, be, seen = rand(B, H), layer.buffers(B), {}
        x.copy_(inp)
        graph.replay()
        eager = inp.clone()
        layer.step(eager, be, B, 1, pos, twin, prefix, P, seen=seen)
        torch.cuda.synchronize()
        assert torch.equal(x, eager) and torch.equal(b["att"], be["att"])
        assert torch.equal(kv.k, twin.k) and torch.equal(kv.v_scale, twin.v_scale)
        check_step(layer, be, seen, B, 1, pos.tolist(), twin, prefix, P, None, f"step {n}")
        pos += 1


def test_an_fp16_cache_quantised_behind_the_existing_prefill(gpu):
    """mt_rope_cache and mt_attention fill an fp16 cache; its copy in 8 bits serves the next step."""
    rng = np.random.default_rng(2)
    M = 21
    qkv = torch.from_numpy(rng.standard_normal((M, (HQ + 2 * HKV) * 64)).astype(np.float32)).to(gpu)
    inv = torch.from_numpy(INV).to(gpu)
    h16 = mt.KV.empty(1, HKV, CAP, torch.float16, gpu)
    mt.rope_cache(qkv, qkv.stride(0), M, HQ, HKV, 0, h16.k, h16.v, CAP, inv)
    f8 = mt.KV.empty(1, HKV, CAP, torch.uint8, gpu)
    mt.kv_copy(h16, f8, 1, M)
    for n in ("k", "v"):
        x = getattr(h16, n).double().cpu().numpy()[0, :, :M]
        assert np.array_equal(values(f8, n)[0, :, :M], U.decode(*U.encode(x, 64), 64))
    q = torch.from_numpy(rng.standard_normal((1, HQ * 64)).astype(np.float32)).to(gpu)
    out = torch.zeros_like(q)
    mt.attention_shared(q, 1, 1, HQ, HKV, torch.tensor([M - 1], dtype=torch.int32, device=gpu), f8, out)
    for h in range(HQ):
        kh = h // (HQ // HKV)
        want, tol = U.attend64(q.double().cpu().numpy()[0].reshape(HQ, 64)[h], values(f8, "k")[0, kh], values(f8, "v")[0, kh], 0, M, 0.125)
        assert np.abs(out.double().cpu().numpy()[0].reshape(HQ, 64)[h] - want).max() <= tol
