"""The paged operators together, as a serving loop uses them: a voice prompt written into pages that many sequences' tables name,
ragged texts behind it, decode steps of the batch, eagerly and as replayed graphs, split keys and their workspaces among them.
Every attention is checked in 64 bits on the cache that stands in the pages."""
import numpy as np
import pytest
import torch

import mingtts as mt
import _f8_util as U
from _gpu_util import say
from _paged_util import TORCH, Case

pytestmark = pytest.mark.gpu
HQ, HKV, PAGE = 14, 2, 16
INV = (1.0 / 1e6 ** (np.arange(32) / 32)).astype(np.float32)


class Server:
    """One layer's cache: B sequences behind a prompt of P slots (whole pages, shared), up to `slots` each."""

    def __init__(self, gpu, kind, B, P, slots, window=0, sinks=0):
        self.gpu, self.kind, self.B, self.P, self.window, self.sinks = gpu, kind, B, P, window, sinks
        n, shared = slots // PAGE, P // PAGE
        order = torch.randperm(shared + B * (n - shared) + 3, generator=torch.Generator().manual_seed(B + P))
        self.table = torch.full((B + 1, n), -1, dtype=torch.int32)
        self.table[:, :shared] = order[:shared]
        self.table[:B, shared:] = order[shared:shared + B * (n - shared)].view(B, -1)
        self.kv = mt.PagedKV.empty(len(order), HKV, PAGE, self.table[:B].to(gpu), TORCH[kind])
        self.prompt = mt.PagedKV(self.kv.k, self.kv.v, self.table[B:].to(gpu), self.kv.k_scale, self.kv.v_scale)
        self.inv = torch.from_numpy(INV).to(gpu)

    def rows(self, n, seed):
        g = torch.Generator(device=self.gpu)
        g.manual_seed(seed)
        return torch.randn(n, (HQ + 2 * HKV) * 64, generator=g, device=self.gpu)

    def layer(self, qkv, B, T, pos, q, out, kv=None, counts=None, **o):
        kv = kv or self.kv
        mt.rope_append_paged(qkv, B, T, HQ, HKV, pos, kv, self.inv, q, counts=counts)
        mt.attention_paged(q, B, T, HQ, HKV, pos, kv, out, counts=counts, window=self.window, sinks=self.sinks, **o)

    def values(self, name, b, n):
        """The slots before n of sequence b as the pages hold them, [hkv, n, 64] in 64 bits."""
        page = self.table[b, :(n + PAGE - 1) // PAGE].long()
        x = getattr(self.kv, name).cpu()[page].transpose(0, 1).reshape(HKV, -1, 64)[:, :n]
        if self.kind != "f8":
            return x.double().numpy()
        s = getattr(self.kv, name + "_scale").cpu()[page].transpose(0, 1).reshape(HKV, -1)[:, :n]
        return U.decode(x.numpy(), s.numpy()[..., None], 64)

    def check(self, qkv, q, out, T, pos, counts=None, b0=0):
        x, qs, o = (t.double().cpu().numpy() for t in (qkv, q, out))
        n = [T] * len(pos) if counts is None else counts
        half = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "f8": 2.0 ** -4}[self.kind]
        for s, p0 in enumerate(pos):
            b = b0 + s
            k, v = self.values("k", b, p0 + n[s]), self.values("v", b, p0 + n[s])
            for t in range(n[s]):
                r, p = s * T + t, p0 + t
                heads = x[r].reshape(-1, 64)
                rot = U.rope64(heads[:HQ + HKV], p, INV)
                assert np.abs(qs[r].reshape(HQ, 64) - rot[:HQ]).max() <= 2.0 ** -24 * np.abs(rot).max() + 1e-14
                # the appended rows: half a step of the value (8 bits: or of the block's least step, 2^-9 of a scale that is at most
                # 2 / 448 of the block's largest value)
                for got, want in ((k[:, p], rot[HQ:]), (v[:, p], heads[HQ + HKV:])):
                    low = np.abs(want).max(-1, keepdims=True) * (2.0 ** -10 * 2 / 448 if self.kind == "f8" else 0)
                    assert (np.abs(got - want) <= half * np.abs(want) + low + (2.0 ** -25 if self.kind == "f16" else 1e-14)).all()
                j = np.arange(p + 1)
                if self.window:
                    j = j[(j > p - self.window) | (j < self.sinks)]
                for h in range(0, HQ, 3):
                    kh = h // (HQ // HKV)
                    want, tol = U.attend64(qs[r].reshape(HQ, 64)[h], k[kh, j], v[kh, j], 0, len(j), 0.125)
                    assert np.abs(o[r].reshape(HQ, 64)[h] - want).max() <= tol, (b, t, h)


@pytest.mark.parametrize("kind", ["f32", "f16", "f8"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 21)])
def test_serving_loop(gpu, kind, window, sinks):
    say(f"serving loop {kind} {window}")
    B, P, T = 3, 48, 20
    s = Server(gpu, kind, B, P, 160, window, sinks)
    i = lambda a: torch.tensor(a, dtype=torch.int32, device=gpu)  # noqa: E731
    z = lambda n: torch.zeros(n, HQ * 64, device=gpu)  # noqa: E731
    # the prompt, once, into the pages that every table begins with
    qkv, q, out = s.rows(P, 1), z(P), z(P)
    s.layer(qkv, 1, P, i([0]), q, out, kv=s.prompt)
    s.check(qkv, q, out, P, [0])
    # ragged texts behind it
    counts = [20, 13, 1]
    qkv, q, out = s.rows(B * T, 2), z(B * T), z(B * T)
    s.layer(qkv, B, T, i([P] * B), q, out, counts=i(counts))
    s.check(qkv, q, out, T, [P] * B, counts)
    # decode steps, eagerly and then replayed from one graph while the positions advance on the device
    pos = i([P + c for c in counts])
    at = [P + c for c in counts]
    qkv, q, out = s.rows(B, 3), z(B), z(B)
    s.layer(qkv, B, 1, pos, q, out)
    s.check(qkv, q, out, 1, at)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        s.layer(qkv, B, 1, pos, q, out)
        pos.add_(1)
    pos.add_(1)
    for step in range(5):
        at = [a + 1 for a in at]
        qkv.copy_(s.rows(B, 10 + step))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert pos.tolist() == [a + 1 for a in at]
        s.check(qkv, q, out, 1, at)
        s.rows(100, step).sum()  # the program's own work between replays


def split_case(gpu, page=16, **o):
    return Case(gpu, "f16", **{**dict(B=2, T=1, hq=14, hkv=2, cap=4096, page=page, pos=[4095, 2000]), **o})


class Call:
    """A case's attention as a program holds it: tensors that stay, outputs of its own."""

    def __init__(self, case, workspace=None):
        self.c, self.ws = case, workspace
        self.q = torch.from_numpy(case.q).to(case.gpu)
        self.pos = torch.tensor(case.pos, dtype=torch.int32, device=case.gpu)
        self.out = torch.zeros(case.B * case.T, case.hq * 64, device=case.gpu)

    def __call__(self, stream=None):
        c = self.c
        f = mt.attention_sinks if c.page is None else mt.attention_paged
        f(self.q, c.B, c.T, c.hq, c.hkv, self.pos, c.kv, self.out, workspace=self.ws, stream=stream)

    def check(self):
        c = self.c
        c.check(self.out.cpu().double().numpy().reshape(c.B, c.T, c.hq, 64))
        self.out.fill_(7.0)


def need(c):
    slots = c.cap if c.page is None else (c.cap + c.page - 1) // c.page * c.page
    return mt.load().mt_attention_window_workspace(c.B, c.T, c.hq, c.hkv, slots, 0, 0, mt.F16)


def test_one_workspace_for_calls_of_many_sizes(gpu):
    """In turn on one stream: what a call leaves in a workspace means nothing to the next, whatever its sizes."""
    calls = [split_case(gpu), split_case(gpu, cap=6000, pos=[5999, 10]), split_case(gpu, page=None, T=3, pos=[4000, 17]),
             split_case(gpu, B=5, pos=[4095, 1, 300, 4000, 64])]
    ws = torch.full((max(need(c) for c in calls),), 0xA5, dtype=torch.uint8, device=gpu)
    assert min(need(c) for c in calls) > 0
    calls = [Call(c, ws) for c in calls]
    for _ in range(3):
        for c in calls:
            c()
        torch.cuda.synchronize()
        for c in calls:
            c.check()


def test_graphs_of_split_keys(gpu):
    """Two graphs that share a workspace, replayed in turn with eager calls and other work between, and one with its own."""
    a, b = split_case(gpu), split_case(gpu, cap=8192, pos=[8191, 5000])
    ws = torch.empty(max(need(a), need(b)), dtype=torch.uint8, device=gpu)
    calls, graphs = [Call(a, ws), Call(b, ws), Call(a)], []
    stream = torch.cuda.Stream()
    for c in calls:
        c()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            c()
            c()
        graphs.append(g)
    for turn in range(4):
        for c, g in zip(calls, graphs):
            c.out.fill_(7.0)
            g.replay()
            torch.cuda.synchronize()
            c.check()
            if turn % 2:
                c()
                torch.cuda.synchronize()
                c.check()


def test_two_streams_at_once(gpu):
    """Calls on two streams, a workspace each (the allocator's, by stream)."""
    calls = [Call(split_case(gpu, seed=s)) for s in range(2)]
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    for _ in range(20):
        for c, s in zip(calls, streams):
            c(stream=s)
    torch.cuda.synchronize()
    for c in calls:
        c.check()


@pytest.mark.parametrize("kind", ["f32", "f16", "f8"])
@pytest.mark.parametrize("T", [1, 300])
def test_pages_and_contiguous_caches_give_the_same_bits(gpu, kind, T):
    """The same slots in pages of several sizes and side by side: one order of sums."""
    out = []
    for page in (None, 16, 64, 128):
        c = Case(gpu, kind, 2, T, 14, 2, 640, page=page, pos=[640 - T, 300], window=200, sinks=20, seed=4)
        out.append(c.run(len_max=640))
    for o in out[1:]:
        assert (o == out[0]).all()
