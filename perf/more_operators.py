"""Timed cases of the paged caches: the step that writes them, the attention that reads them, and attention
in a sliding window with first positions that stay visible, over pages and over contiguous caches.

A paged cache keeps the keys and values of many sequences in one pool of pages, [pages, hkv, page, 64] each; slot s of
sequence b is row s % page of pool page table[b, s // page].  A table entry outside the pool is no page: what a sequence has
not reached yet, or what its window has left behind and the server has taken back.

Kinds of case (each dict's "kind"):

  append  the step that writes a paged cache: RoPE of the query and key heads of T new rows for each of B sequences
          at positions offset + pos[b] + t, the rotated keys and the values stored at slots pos[b] + t in the cache's type.
          Sequence b has counts[b] <= T rows.  8-bit caches hold e4m3 codes and one scale byte s a head and slot that
          stands for 2^(s - 127), the least power of two, 2^-126 or more, that brings the 64 values within 448.
  paged   attention of such rows over their sequences' pages up to their own slot, grouped query heads; with a window,
          over the last `window` slots and the first `sinks` ones.
  sinks   the same over contiguous caches [B, hkv, cap, 64].

Heads are 64 wide; 14 query and 2 key heads, caches of 512 positions and a voice prompt of 174 are the backbone's, the other
sizes are generic.  Activations are N(0, 1).
"""
import math
import os
import sys

import torch

own = False

HQ, HKV, D = 14, 2, 64
SCALE = 0.125
TYPES = {"f8": torch.uint8, "f16": torch.float16, "f32": torch.float32}
NONE = -1  # a table entry that is no page


def listed():
    heads = dict(hq=HQ, hkv=HKV)
    return [
        # One decode step's cache write for the guided pair of one utterance: the smallest call.
        dict(name="append_step_2", kind="append", B=2, T=1, **heads, cap=512, page=16, cache="f16", offset=0),
        # Texts of many utterances written in 8 bits behind a voice prompt of 174 positions.
        dict(name="append_prompts_16", kind="append", B=16, T=330, **heads, cap=512, page=64, cache="f8", offset=174),
        # The guided pair's attention within 512 positions: latency.
        dict(name="paged_step_2", kind="paged", B=2, T=1, **heads, cap=512, page=16, cache="f16", window=0, sinks=0),
        # Batched serving, sequences of all lengths up to a long one, small pages: the bytes of the caches.
        dict(name="paged_step_64", kind="paged", B=64, T=1, **heads, cap=4096, page=16, cache="f16", window=0, sinks=0),
        # A full server in 8 bits.
        dict(name="paged_step_f8_128", kind="paged", B=128, T=1, **heads, cap=4096, page=64, cache="f8", window=0, sinks=0),
        # The largest batch: more bytes than any cache on the chip holds.
        dict(name="paged_step_256", kind="paged", B=256, T=1, **heads, cap=4096, page=32, cache="f16", window=0, sinks=0),
        # One sequence with a very long cache: few rows, the keys are split.
        dict(name="paged_long_1", kind="paged", B=1, T=1, **heads, cap=131072, page=256, cache="f16", window=0, sinks=0),
        # Streams far past their window that keep the voice prompt in sight; the pages between are given back.
        dict(name="paged_window_96", kind="paged", B=96, T=1, **heads, cap=16384, page=64, cache="f8", window=1024, sinks=174),
        # Ragged texts attended in one call behind what their sequences hold already.
        dict(name="paged_prompts_8", kind="paged", B=8, T=130, **heads, cap=1280, page=16, cache="f16", window=0, sinks=0),
        # Streams in contiguous caches, window and voice prompt.
        dict(name="sinks_step_32", kind="sinks", B=32, T=1, **heads, cap=8192, cache="f16", window=512, sinks=174),
        # A long prompt in a window: products.
        dict(name="sinks_prompt_4096", kind="sinks", B=1, T=4096, **heads, cap=4096, cache="f16", window=1024, sinks=64),
        # Ragged prompts over fp32 caches, another head layout, odd sizes.
        dict(name="sinks_prompts_4_f32", kind="sinks", B=4, T=701, hq=12, hkv=4, cap=1003, cache="f32", window=301, sinks=51),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, its logarithm uniform."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "paged", "paged", "sinks"])
    hq, hkv = rng.choice([(14, 2), (14, 2), (16, 16), (8, 2), (12, 4), (16, 1)])
    cache = rng.choice(["f16", "f16", "f8", "f32"])
    c = dict(kind=kind, hq=hq, hkv=hkv, cache=cache)
    if kind != "sinks":
        c["page"] = rng.choice([16, 16, 32, 48, 64, 128, 256])
    if kind == "append":
        c["B"] = _spread(rng, 1, 256)
        c["T"] = _spread(rng, 1, max(1, 5000 // c["B"]))
        c["cap"] = c["T"] + _spread(rng, 4, 2000)
        c["offset"] = _spread(rng, 1, 4000) - 1
        return c
    c["B"] = _spread(rng, 1, 128)
    c["T"] = 1 if rng.random() < 0.6 else _spread(rng, 2, max(2, 1500 // c["B"]))
    room = max(64, (400000 if c["T"] == 1 else 200000) // (c["B"] * hkv))
    c["cap"] = max(c["T"], _spread(rng, 16, min(room, 60000 if c["T"] == 1 else 6000)))
    c["window"] = 0 if rng.random() < (0.6 if kind == "paged" else 0.2) else _spread(rng, 1, 2000)
    c["sinks"] = _spread(rng, 1, 300) - 1 if c["window"] else 0
    if kind == "sinks" and cache == "f8":
        c["cap"] = (c["cap"] + 3) // 4 * 4
    return c


# --------------------------------------------------------------- inputs --

def _cache(g, shape, kind):
    """Keys or values of a cache: the tensor in the cache's type, and its scales."""
    x = torch.randn(*shape, D, generator=g, device="cuda")
    if kind != "f8":
        return x.to(TYPES[kind]), None
    s = ((x.abs().amax(-1, keepdim=True).view(torch.int32) + 0x1FFFFF) >> 23) - 8  # 448 = 1.75 2^8
    code = (x * ((254 - s) << 23).view(torch.float32)).to(torch.float8_e4m3fn).view(torch.uint8)
    return code, s[..., 0].to(torch.uint8).contiguous()


def _pages(c):
    """Table entries a sequence, and pages of the pool (some are nobody's)."""
    n = (c["cap"] + c["page"] - 1) // c["page"]
    return n, c["B"] * n + 7


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    c = dict(case)
    B, T, hq, hkv, cap = c["B"], c["T"], c["hq"], c["hkv"], c["cap"]
    st = {"case": c}
    # The rows a sequence brings: all T for a decode step, ragged for prompts; the slots before them are filled to any
    # length the cache has room for (the first sequence fills it).
    counts = torch.randint(max(1, T // 2), T + 1, (B,), generator=g, device="cuda")
    counts[0] = T
    pos = (torch.rand(B, generator=g, device="cuda") * (cap - T + 1)).long().clamp(0, cap - T)
    pos[0] = cap - T
    st["pos"], st["counts"] = pos.to(torch.int32), counts.to(torch.int32) if T > 1 else None
    if "page" in c:
        n, pool = _pages(c)
        table = torch.randperm(pool, generator=g, device="cuda")[:B * n].view(B, n)
        first = torch.arange(n, device="cuda") * c["page"]
        gone = first >= (pos + counts)[:, None]
        if c.get("window"):  # pages that no row sees any more are taken back
            gone |= (first >= c["sinks"]) & (first + c["page"] <= (pos + 1 - c["window"])[:, None])
        st["table"] = torch.where(gone, NONE, table).to(torch.int32)
        shape = (pool, hkv, c["page"])
    else:
        shape = (B, hkv, cap)
    if c["kind"] == "append":
        st["qkv"] = torch.randn(B * T, (hq + 2 * hkv) * D, generator=g, device="cuda")
        st["inv_freq"] = (1.0 / 1e6 ** (torch.arange(32, device="cuda", dtype=torch.float64) / 32)).float()
        st["k"] = torch.zeros(*shape, D, dtype=TYPES[c["cache"]], device="cuda")
        st["k_scale"] = torch.ones(shape, dtype=torch.uint8, device="cuda") if c["cache"] == "f8" else None
        st["v"] = torch.zeros_like(st["k"])
        st["v_scale"] = torch.ones_like(st["k_scale"]) if c["cache"] == "f8" else None
        st["q"] = torch.zeros(B * T, hq * D, device="cuda")
        return st
    st["q"] = torch.randn(B * T, hq * D, generator=g, device="cuda")
    st["k"], st["k_scale"] = _cache(g, shape, c["cache"])
    st["v"], st["v_scale"] = _cache(g, shape, c["cache"])
    st["out"] = torch.zeros(B * T, hq * D, device="cuda")
    return st


# ------------------------------------------------------------------ run --

def run(st):
    c = st["case"]
    if own:
        if "mt" not in st:  # the handle a program keeps beside its caches
            st["mt"] = mt = _mt()
            kv = (st["k"], st["v"], st["k_scale"], st["v_scale"])
            st["kv"] = mt.PagedKV(*kv[:2], st["table"], *kv[2:]) if "page" in c else mt.KV(*kv)
        return {"append": _own_append, "paged": _own_paged, "sinks": _own_sinks}[c["kind"]](st, c)
    return _plain_append(st, c) if c["kind"] == "append" else _plain_attend(st, c)


def _mt():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ming-tts_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import mingtts
    return mingtts


def _own_append(st, c):
    st["mt"].rope_append_paged(st["qkv"], c["B"], c["T"], c["hq"], c["hkv"], st["pos"], st["kv"], st["inv_freq"], st["q"],
                               counts=st["counts"], offset=c["offset"])
    return _written(st, c)


def _own_paged(st, c):
    st["mt"].attention_paged(st["q"], c["B"], c["T"], c["hq"], c["hkv"], st["pos"], st["kv"], st["out"], counts=st["counts"],
                             window=c["window"], sinks=c["sinks"], scale=SCALE)
    return st["out"]


def _own_sinks(st, c):
    st["mt"].attention_sinks(st["q"], c["B"], c["T"], c["hq"], c["hkv"], st["pos"], st["kv"], st["out"], counts=st["counts"],
                             window=c["window"], sinks=c["sinks"], scale=SCALE)
    return st["out"]


def _written(st, c):
    """The rotated queries and the pools; 8-bit ones as the values of their codes and of their scale bytes."""
    out = {"q": st["q"]}
    for n in ("k", "v"):
        out[n] = st[n].view(torch.float8_e4m3fn) if c["cache"] == "f8" else st[n]
        if c["cache"] == "f8":
            out[n + "_scale"] = st[n + "_scale"].view(torch.float8_e8m0fnu)
    return out


def _rows(st, c):
    """[B, T]: the rows' own slots, and whether the sequence has the row."""
    t = torch.arange(c["T"], device="cuda")
    slot = st["pos"].long()[:, None] + t
    if st["counts"] is None:
        return slot, torch.ones_like(slot, dtype=torch.bool)
    return slot, t < st["counts"].long()[:, None]


def _nearest(x, bits, least):
    """x (64 bits) to `bits` bits behind the leading one, ties to even, steps no finer than 2^least."""
    step = torch.ldexp(torch.ones_like(x), (torch.frexp(x)[1] - 1 - bits).clamp_min(least))
    return torch.round(x / step) * step


def _plain_append(st, c):
    B, T, hq, hkv, L = c["B"], c["T"], c["hq"], c["hkv"], c["page"]
    slot, has = _rows(st, c)
    ang = (slot + c["offset"]).double().unsqueeze(-1) * st["inv_freq"].double()  # [B, T, 32]
    cos, sin = ang.cos()[:, :, None], ang.sin()[:, :, None]
    x = st["qkv"].view(B, T, hq + 2 * hkv, D).double()
    lo, hi = x[:, :, :hq + hkv, :32], x[:, :, :hq + hkv, 32:]
    rot = torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1)
    q = rot[:, :, :hq].reshape(B, T, -1).float()
    st["q"].copy_(torch.where(has[..., None], q, st["q"].view(B, T, -1)).view(B * T, -1))
    b, t = has.nonzero(as_tuple=True)
    at = slot[b, t]
    page, row = st["table"].long()[b, at // L], at % L
    for name, rows in (("k", rot[:, :, hq:]), ("v", x[:, :, hq + hkv:])):
        r = rows[b, t]  # [n, hkv, 64]
        if c["cache"] == "f32":
            st[name][page, :, row] = r.float()
        elif c["cache"] == "f16":
            st[name][page, :, row] = _nearest(r, 10, -24).half()
        else:
            m, e = torch.frexp(r.abs().amax(-1, keepdim=True))
            e = (e - 9 + (m > 0.875)).clamp_min(-126)  # top <= 448 2^e = 0.875 2^(e + 9)
            st[name][page, :, row] = _nearest(torch.ldexp(r, -e), 3, -9).float().to(torch.float8_e4m3fn).view(torch.uint8)
            st[name + "_scale"][page, :, row] = (e[..., 0] + 127).to(torch.uint8)
    return _written(st, c)


def _contiguous(st, c, name):
    """A sequence's keys or values side by side in fp32, [B, hkv, slots, 64]."""
    x = st[name].view(torch.float8_e4m3fn) if c["cache"] == "f8" else st[name]
    s = st[name + "_scale"]
    if "page" in c:
        page = st["table"].long().clamp_min(0)
        x = x.view(torch.uint8)[page].view(x.dtype) if c["cache"] == "f8" else x[page]
        x = x.transpose(1, 2).flatten(2, 3)
        s = None if s is None else s[page].transpose(1, 2).flatten(2, 3)
    x = x.float()
    return x if s is None else x * (s.int() << 23).view(torch.float32).unsqueeze(-1)


def _plain_attend(st, c):
    B, T, hq, hkv, G = c["B"], c["T"], c["hq"], c["hkv"], c["hq"] // c["hkv"]
    k, v = _contiguous(st, c, "k"), _contiguous(st, c, "v")
    q = st["q"].view(B, T, hkv, G, D).permute(0, 2, 1, 3, 4)  # [B, hkv, T, G, 64]
    slot, has = _rows(st, c)
    j = torch.arange(k.shape[2], device="cuda")
    ok = j <= slot[..., None]  # [B, T, slots]
    if c["window"]:
        ok &= (j > slot[..., None] - c["window"]) | (j < c["sinks"])
    s = torch.matmul(q.reshape(B, hkv, T * G, D), k.transpose(-1, -2).contiguous()).view(B, hkv, T, G, -1)
    s = torch.where(ok[:, None, :, None], s * SCALE, -math.inf)
    e = torch.exp(s - s.amax(-1, keepdim=True))
    o = torch.matmul(e.view(B, hkv, T * G, -1), v).view(B, hkv, T, G, D)
    o = (o / e.sum(-1, keepdim=True)).permute(0, 2, 1, 3, 4).reshape(B, T, hq * D)
    return torch.where(has[..., None], o, st["out"].view(B, T, -1)).view(B * T, -1)


# ----------------------------------------------------------------- work --

def work(case):
    c = case
    B, T, hq, hkv = c["B"], c["T"], c["hq"], c["hkv"]
    # The first sequence brings all T rows and fills the cache; the others bring T / 2 to T behind 0 to cap - T filled slots.
    n = T if T == 1 else 0.75 * T
    rows = T + (B - 1) * n
    row = {"f8": 65, "f16": 128, "f32": 256}[c["cache"]]
    if c["kind"] == "append":
        return {"bytes": rows * ((hq + 2 * hkv) * 256 + hq * 256 + hkv * 2 * row), "flops": rows * (hq + hkv) * 32 * 6}

    def visible(last):
        w = c["window"]
        return last if not w or last <= w else w + min(c["sinks"], last - w)

    def sequence(filled, n):  # keys that its rows see, summed and together
        return (n * sum(visible(filled + n * (i + 0.5) / 8) for i in range(8)) / 8,
                min(filled + n, visible(filled + n) + (n - 1 if c["window"] else 0)))

    pairs, keys = sequence(c["cap"] - T, T)
    for i in range(64):
        p, k = sequence((c["cap"] - T) * (i + 0.5) / 64, n)
        pairs, keys = pairs + p * (B - 1) / 64, keys + k * (B - 1) / 64
    return {"bytes": 2 * hkv * row * keys + rows * hq * D * 8 + (4 * keys / c["page"] if "page" in c else 0),
            "flops": 4 * D * hq * pairs}


# ---------------------------------------------------------------- exact --

def _value64(code, s):
    """The values that codes and scale bytes stand for, in 64 bits, from the bits of the format."""
    c = code.to(torch.int64)
    m, e = c & 7, (c >> 3) & 15
    v = torch.where(e > 0, (8 + m).double() * 2.0 ** (e - 10).double(), m.double() * 2.0 ** -9)
    return torch.where(c > 127, -v, v) * 2.0 ** (s.double().unsqueeze(-1) - 127)


def _block64(x):
    """x [..., 64]: the scaled values rounded to e4m3, and the scales, in 64 bits."""
    top = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(top.clamp_min(1e-300) / 448))
    e = torch.where(448 * 2.0 ** e < top, e + 1, torch.where(448 * 2.0 ** (e - 1) >= top, e - 1, e)).clamp_min(-126.0)
    z = x * 2.0 ** -e
    step = 2.0 ** (torch.floor(torch.log2(z.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(z / step) * step, 2.0 ** e[..., 0]


def exact(case, seed):
    st, c = prepare(case, seed), case
    B, T, hq, hkv, G = c["B"], c["T"], c["hq"], c["hkv"], c["hq"] // c["hkv"]
    pos = st["pos"].tolist()
    n = [T] * B if st["counts"] is None else st["counts"].tolist()
    f8 = c["cache"] == "f8"
    if c["kind"] == "append":
        out = {"q": st["q"].double(), "k": st["k"].double(), "v": st["v"].double()}
        if f8:
            out.update(k_scale=2.0 ** (st["k_scale"].double() - 127), v_scale=2.0 ** (st["v_scale"].double() - 127))
        x = st["qkv"].double().view(B, T, hq + 2 * hkv, D)
        for b in range(B):
            p = torch.arange(pos[b], pos[b] + n[b], device="cuda")
            w = torch.outer((p + c["offset"]).double(), st["inv_freq"].double())
            turn = torch.polar(torch.ones_like(w), w)[:, None]
            z = torch.complex(x[b, :n[b], :hq + hkv, :32].contiguous(), x[b, :n[b], :hq + hkv, 32:].contiguous()) * turn
            z = torch.cat([z.real, z.imag], -1)
            out["q"].view(B, T, hq, D)[b, :n[b]] = z[:, :hq]
            page, row = st["table"][b].long()[p // c["page"]], p % c["page"]
            for name, y in (("k", z[:, hq:]), ("v", x[b, :n[b], hq + hkv:])):
                if f8:
                    y, s = _block64(y)
                    out[name + "_scale"][page, :, row] = s
                out[name][page, :, row] = y
        return out
    out = st["out"].double()
    for b in range(B):
        ln = pos[b] + n[b]
        j = torch.arange(ln, device="cuda")
        if c["window"]:  # what some row sees
            j = j[(j > pos[b] - c["window"]) | (j < c["sinks"])]
        kv = []
        for name in ("k", "v"):
            if "page" in c:
                at = (st["table"][b].long()[j // c["page"]], slice(None), j % c["page"])
                r = _value64(st[name][at], st[name + "_scale"][at]) if f8 else st[name][at].double()  # [keys, hkv, 64]
                kv.append(r.transpose(0, 1).contiguous())
            else:
                kv.append(_value64(st[name][b][:, j], st[name + "_scale"][b][:, j]) if f8 else st[name][b][:, j].double())
        k, v = kv
        kt = k.transpose(1, 2).contiguous()
        for t0 in range(0, n[b], 512):
            t1 = min(n[b], t0 + 512)
            q = st["q"].double().view(B, T, hkv, G, D)[b, t0:t1].permute(1, 2, 0, 3).reshape(hkv, -1, D).contiguous()
            s = (q @ kt).view(hkv, G, t1 - t0, -1) * SCALE
            row = torch.arange(pos[b] + t0, pos[b] + t1, device="cuda")[:, None]
            hide = j[None] > row
            if c["window"]:
                hide |= (j[None] <= row - c["window"]) & (j[None] >= c["sinks"])
            p = torch.softmax(s.masked_fill(hide, -math.inf), -1)
            o = (p.reshape(hkv, -1, len(j)) @ v).view(hkv, G, t1 - t0, D)
            out.view(B, T, hkv, G, D)[b, t0:t1] = o.permute(2, 0, 1, 3)
    return out
