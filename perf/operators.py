"""Timed cases of the 8-bit operators: caches and weights held in e4m3 with power-of-two scales,
and the attention of a batch that shares a prefix.

The format.  A block of values x is held as e4m3 codes c (4 exponent bits, 3 mantissa bits, largest
448, no infinities) and one scale byte s that stands for 2^(s - 127): the least power of two, 2^-126
or more, at which the block's largest |x| is at most 448.  x / 2^(s - 127) is rounded to nearest, ties
to even.  A block is the 64 values of one key or value head of a position in a cache, and 128
consecutive values of a row in a matrix (the last block of a row may be shorter).

Kinds of case (each dict's "kind"):

  append  the step that writes a cache: RoPE of the query and key heads of T new rows for each of B
          sequences, the key and value rows appended in 8 bits, and the rows read back as fp16.
          Row t of sequence b stands at slot pos[b] + t and is rotated at the angle of position
          offset + pos[b] + t (the shared prefix comes first); sequence b has counts[b] <= T rows.
  attend  attention of those rows over prefix_len keys that all sequences share and then over the
          sequence's own keys up to the row's, grouped query heads, with an optional window.
  linear  y = epilogue(x w^T) with w in 8 bits and x quantised in blocks of 128 on the way in.

Heads are 64 wide; 14 query and 2 key heads, hidden 896, MLP 4864 and caches of 512 positions are the
backbone's, the other sizes are generic.  Activations are N(0, 1), weights N(0, 0.02^2).
"""
import math
import os
import sys

import torch

own = False

HQ, HKV, D = 14, 2, 64
SCALE = 0.125
TYPES = {"f8": torch.uint8, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # One decode step's cache write for the guided pair of one utterance: the smallest call.
        dict(name="append_step_2", kind="append", B=2, T=1, hq=HQ, hkv=HKV, cap=512, offset=0),
        # Texts of many utterances written behind a shared voice prompt of 174 positions.
        dict(name="append_prompts_16", kind="append", B=16, T=330, hq=HQ, hkv=HKV, cap=512, offset=174),
        # The guided pair's attention in the benchmark's 512-position cache: latency.
        dict(name="attend_step_2", kind="attend", B=2, T=1, hq=HQ, hkv=HKV, cap=512, prefix=0, window=0, cache="f8"),
        # Batched serving, sequences of all lengths up to a long cache: the bytes of the caches.
        dict(name="attend_step_64", kind="attend", B=64, T=1, hq=HQ, hkv=HKV, cap=4096, prefix=0, window=0, cache="f8"),
        # Many utterances of one voice: a long prompt held once, short continuations.
        dict(name="attend_shared_128", kind="attend", B=128, T=1, hq=HQ, hkv=HKV, cap=512, prefix=2048, window=0,
             cache="f8"),
        # The benchmark's 174-position prompt shared by a small batch, in the fp16 caches.
        dict(name="attend_shared_f16_32", kind="attend", B=32, T=1, hq=HQ, hkv=HKV, cap=320, prefix=174, window=0,
             cache="f16"),
        # Their texts' prompts, ragged, attended in one call behind the shared prefix.
        dict(name="attend_prompts_8", kind="attend", B=8, T=130, hq=HQ, hkv=HKV, cap=256, prefix=1000, window=0,
             cache="f8"),
        # One sequence with a very long cache: few rows, the keys are split.
        dict(name="attend_long_1", kind="attend", B=1, T=1, hq=HQ, hkv=HKV, cap=131072, prefix=0, window=0, cache="f8"),
        # gate|up of one decode step of the guided pair, fp32 activations.
        dict(name="linear_step_2", kind="linear", M=2, N=4864, K=896, gated=True, bias=False, gelu=False),
        # down of a decode step for a batch of sixteen.
        dict(name="linear_down_16", kind="linear", M=16, N=896, K=4864, gated=False, bias=False, gelu=False),
        # gate|up of a prompt that fills the backbone's cache.
        dict(name="linear_prompt_512", kind="linear", M=512, N=4864, K=896, gated=True, bias=False, gelu=False),
        # A large generic product: bias and GELU behind 4096 rows.
        dict(name="linear_4096", kind="linear", M=4096, N=4096, K=4096, gated=False, bias=True, gelu=True),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, its logarithm uniform."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "linear"])
    hq, hkv = rng.choice([(14, 2), (14, 2), (16, 16), (8, 2), (12, 4), (16, 1)])
    if kind == "append":
        B = _spread(rng, 1, 48)
        T = _spread(rng, 1, max(1, 6000 // B))
        return dict(kind="append", B=B, T=T, hq=hq, hkv=hkv, cap=(T + _spread(rng, 4, 2000) + 3) // 4 * 4,
                    offset=_spread(rng, 1, 4000) - 1)
    if kind == "attend":
        cache = rng.choice(["f8", "f8", "f8", "f16", "f32"])
        B = _spread(rng, 1, 96)
        T = 1 if rng.random() < 0.6 else _spread(rng, 2, max(2, 700 // B))
        cap = (max(T, min(_spread(rng, 16, 4096), 200000 // B)) + 3) // 4 * 4
        prefix = 0 if rng.random() < 0.3 else _spread(rng, 1, 4000)
        window = 0 if rng.random() < 0.8 else _spread(rng, 1, 600)
        return dict(kind="attend", B=B, T=T, hq=hq, hkv=hkv, cap=cap, prefix=prefix, window=window, cache=cache)
    M = _spread(rng, 1, 3000)
    N = _spread(rng, 16, 4800)
    K = 16 * _spread(rng, 4, 256)
    gated = rng.random() < 0.4
    return dict(kind="linear", M=M, N=N, K=K, gated=gated, bias=rng.random() < 0.5, gelu=not gated and rng.random() < 0.3)


# --------------------------------------------------------------- inputs --

def _pow2(byte):
    """2^(s - 127) of scale bytes 1 .. 254, exactly."""
    return (byte.to(torch.int32) << 23).view(torch.float32)


def _encode(x, width):
    """fp32 [..., n] in blocks of `width` along the last axis (n a multiple of it): codes and scale bytes."""
    b = x.reshape(*x.shape[:-1], -1, width)
    top = b.abs().amax(-1)
    s = (((top.view(torch.int32) + 0x1FFFFF) >> 23) - 8).clamp_min(1)
    code = (b * _pow2(254 - s).unsqueeze(-1)).to(torch.float8_e4m3fn)
    return code.view(torch.uint8).reshape(x.shape), s.to(torch.uint8)


def _decode(code, s, width):
    v = code.view(torch.float8_e4m3fn).to(torch.float32)
    return (v.reshape(*v.shape[:-1], -1, width) * _pow2(s).unsqueeze(-1)).reshape(v.shape)


def _matrix(w):
    """A weight matrix in 8 bits: codes [N, K] and scales [N, 4 ceil(K / 512)], rows padded with zeros."""
    n, k = w.shape
    code, s = _encode(torch.nn.functional.pad(w, (0, -k % 128)), 128)
    return code[:, :k].contiguous(), torch.nn.functional.pad(s, (0, -s.shape[1] % 4)).contiguous()


def _cache(g, shape, kind):
    """Keys or values of a cache: the tensor in the cache's type, and its scales."""
    x = torch.randn(*shape, D, generator=g, device="cuda")
    if kind != "f8":
        return x.to(TYPES[kind]), None
    code, s = _encode(x, D)
    return code, s.reshape(shape).contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    c = dict(case)
    st = {"case": c}
    if c["kind"] == "linear":
        M, N, K = c["M"], c["N"], c["K"]
        st["x"] = torch.randn(M, K, generator=g, device="cuda")
        st["w"] = _matrix(torch.randn(N, K, generator=g, device="cuda") * 0.02)
        st["w2"] = _matrix(torch.randn(N, K, generator=g, device="cuda") * 0.02) if c["gated"] else None
        st["bias"] = torch.randn(N, generator=g, device="cuda").to(torch.float16) if c["bias"] else None
        st["y"] = torch.zeros(M, N, device="cuda")
        return st
    B, T, hq, hkv, cap = c["B"], c["T"], c["hq"], c["hkv"], c["cap"]
    # The rows a sequence brings: all T for a decode step, ragged for prompts; the slots before them
    # are filled to any length the cache has room for (the first sequence fills it).
    counts = torch.randint(max(1, T // 2), T + 1, (B,), generator=g, device="cuda")
    counts[0] = T
    pos = (torch.rand(B, generator=g, device="cuda") * (cap - T + 1)).long().clamp(0, cap - T)
    pos[0] = cap - T
    st["pos"], st["counts"] = pos.to(torch.int32), counts.to(torch.int32) if T > 1 else None
    if c["kind"] == "append":
        st["qkv"] = torch.randn(B * T, (hq + 2 * hkv) * D, generator=g, device="cuda")
        st["inv_freq"] = (1.0 / 1e6 ** (torch.arange(32, device="cuda", dtype=torch.float64) / 32)).float()
        st["k"], st["k_scale"] = torch.zeros(B, hkv, cap, D, dtype=torch.uint8, device="cuda"), torch.ones(
            B, hkv, cap, dtype=torch.uint8, device="cuda")
        st["v"], st["v_scale"] = torch.zeros_like(st["k"]), torch.ones_like(st["k_scale"])
        st["q"] = torch.zeros(B * T, hq * D, device="cuda")
        st["k16"] = torch.zeros(B, hkv, cap, D, dtype=torch.float16, device="cuda")
        st["v16"] = torch.zeros_like(st["k16"])
        return st
    st["q"] = torch.randn(B * T, hq * D, generator=g, device="cuda")
    st["k"], st["k_scale"] = _cache(g, (B, hkv, cap), c["cache"])
    st["v"], st["v_scale"] = _cache(g, (B, hkv, cap), c["cache"])
    if c["prefix"]:
        p4 = (c["prefix"] + 3) // 4 * 4
        st["pk"], st["pk_scale"] = _cache(g, (hkv, p4), c["cache"])
        st["pv"], st["pv_scale"] = _cache(g, (hkv, p4), c["cache"])
    st["out"] = torch.zeros(B * T, hq * D, device="cuda")
    return st


# ------------------------------------------------------------------ run --

def run(st):
    c = st["case"]
    if own:
        return {"append": _own_append, "attend": _own_attend, "linear": _own_linear}[c["kind"]](st, c)
    return {"append": _plain_append, "attend": _plain_attend, "linear": _plain_linear}[c["kind"]](st, c)


def _mt():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ming-tts_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import mingtts
    return mingtts


def _own_append(st, c):
    if "mt" not in st:  # the handles a program keeps beside its caches
        st["mt"] = mt = _mt()
        st["kv"] = mt.KV(st["k"], st["v"], st["k_scale"], st["v_scale"])
        st["kv16"] = mt.KV(st["k16"], st["v16"])
    mt = st["mt"]
    mt.rope_append(st["qkv"], c["B"], c["T"], c["hq"], c["hkv"], st["pos"], st["kv"], st["inv_freq"], st["q"],
                   counts=st["counts"], offset=c["offset"])
    mt.kv_copy(st["kv"], st["kv16"], c["B"], c["T"], pos=st["pos"], counts=st["counts"])
    return {"q": st["q"], "k": st["k16"], "v": st["v16"]}


def _own_attend(st, c):
    if "mt" not in st:
        st["mt"] = mt = _mt()
        st["kv"] = mt.KV(st["k"], st["v"], st["k_scale"], st["v_scale"])
        st["prefix"] = mt.KV(st["pk"], st["pv"], st["pk_scale"], st["pv_scale"]) if c["prefix"] else None
    st["mt"].attention_shared(st["q"], c["B"], c["T"], c["hq"], c["hkv"], st["pos"], st["kv"], st["out"],
                              prefix=st["prefix"], prefix_len=c["prefix"], counts=st["counts"], window=c["window"],
                              scale=SCALE)
    return st["out"]


def _own_linear(st, c):
    if "mt" not in st:
        st["mt"] = mt = _mt()
        st["w8"] = mt.F8Matrix(*st["w"])
        st["w28"] = mt.F8Matrix(*st["w2"]) if c["gated"] else None
    F = st["mt"].GemvFlags
    flags = (F.siluGate if c["gated"] else 0) | (F.gelu if c["gelu"] else 0)
    st["mt"].linear_f8(st["x"], st["w8"], st["y"], flags=flags, w2=st["w28"], bias=st["bias"])
    return st["y"]


def _rows(st, c):
    """[B, T]: the rows' own slots, and whether the sequence has the row."""
    t = torch.arange(c["T"], device="cuda")
    slot = st["pos"].long()[:, None] + t
    if st["counts"] is None:
        return slot, torch.ones_like(slot, dtype=torch.bool)
    return slot, t < st["counts"].long()[:, None]


def _plain_append(st, c):
    B, T, hq, hkv = c["B"], c["T"], c["hq"], c["hkv"]
    slot, has = _rows(st, c)
    ang = (slot + c["offset"]).double().unsqueeze(-1) * st["inv_freq"].double()  # [B, T, 32]
    cos, sin = ang.cos().float()[:, :, None], ang.sin().float()[:, :, None]
    x = st["qkv"].view(B, T, hq + 2 * hkv, D)
    lo, hi = x[:, :, :hq + hkv, :32], x[:, :, :hq + hkv, 32:]
    rot = torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1)
    st["q"].copy_(torch.where(has[..., None], rot[:, :, :hq].reshape(B, T, -1), st["q"].view(B, T, -1)).view(B * T, -1))
    b, t = has.nonzero(as_tuple=True)
    at = slot[b, t]
    for name, rows in (("k", rot[:, :, hq:]), ("v", x[:, :, hq + hkv:])):
        code, s = _encode(rows[b, t], D)  # [n, hkv, 64], [n, hkv, 1]
        st[name][b, :, at] = code
        st[name + "_scale"][b, :, at] = s[..., 0]
        st[name + "16"][b, :, at] = _decode(code, s, D).to(torch.float16)
    return {"q": st["q"], "k": st["k16"], "v": st["v16"]}


def _plain_attend(st, c):
    B, T, hq, hkv, P, G = c["B"], c["T"], c["hq"], c["hkv"], c["prefix"], c["hq"] // c["hkv"]
    value = lambda n: _decode(st[n], st[n + "_scale"].unsqueeze(-1), D) if c["cache"] == "f8" else st[n].float()  # noqa: E731
    q = st["q"].view(B, T, hkv, G, D).permute(0, 2, 1, 3, 4)  # [B, hkv, T, G, 64]
    k, v = value("k"), value("v")  # [B, hkv, cap, 64]
    slot, has = _rows(st, c)
    j = torch.arange(P + c["cap"], device="cuda")
    last = P + slot
    ok = j <= last[..., None]  # [B, T, P + cap]
    if c["window"]:
        ok &= j > last[..., None] - c["window"]
    s = torch.matmul(q.reshape(B, hkv, T * G, D), k.transpose(-1, -2)).view(B, hkv, T, G, -1)
    if P:
        pk, pv = value("pk")[:, :P], value("pv")[:, :P]  # [hkv, P, 64]
        rows = q.transpose(0, 1).reshape(hkv, B * T * G, D)
        sp = torch.matmul(rows, pk.transpose(-1, -2)).view(hkv, B, T, G, P).transpose(0, 1)
        s = torch.cat([sp, s], -1)
    s = torch.where(ok[:, None, :, None], s * SCALE, -math.inf)
    e = torch.exp(s - s.amax(-1, keepdim=True))
    o = torch.matmul(e[..., P:].reshape(B, hkv, T * G, -1), v).view(B, hkv, T, G, D)
    if P:
        rows = e[..., :P].transpose(0, 1).reshape(hkv, B * T * G, P)
        o = o + torch.matmul(rows, pv).view(hkv, B, T, G, D).transpose(0, 1)
    o = (o / e.sum(-1, keepdim=True)).permute(0, 2, 1, 3, 4).reshape(B, T, hq * D)
    return torch.where(has[..., None], o, st["out"].view(B, T, -1)).view(B * T, -1)


def _plain_linear(st, c):
    K = c["K"]
    pad = (0, -K % 128)
    x = _decode(*_encode(torch.nn.functional.pad(st["x"], pad), 128), 128)[:, :K]

    def weight(m):
        code, s = m
        s = s[:, :(K + 127) // 128]
        return _decode(torch.nn.functional.pad(code, pad), s, 128)[:, :K]

    y = x @ weight(st["w"]).T
    if c["bias"]:
        y = y + st["bias"].float()
    if c["gated"]:
        y = y / (1 + torch.exp(-y)) * (x @ weight(st["w2"]).T)
    if c["gelu"]:
        y = 0.5 * y * (1 + torch.tanh(0.7978845608028654 * (y + 0.044715 * y * y * y)))
    return y


# ----------------------------------------------------------------- work --

def work(case):
    c = case
    if c["kind"] == "linear":
        M, N, K = c["M"], c["N"], c["K"]
        mats = 2 if c["gated"] else 1
        return {"bytes": 4 * M * K + mats * N * (K + (K + 127) // 128) + (2 * N if c["bias"] else 0) + 4 * M * N,
                "flops": 2 * M * N * K * mats}
    B, T, hq, hkv = c["B"], c["T"], c["hq"], c["hkv"]
    rows = B * (T if T == 1 else 0.75 * T)  # a ragged call's counts are T / 2 to T
    if c["kind"] == "append":
        # qkv read, q written, the rows written in 8 bits, read back and written in 16.
        return {"bytes": rows * ((hq + 2 * hkv) * 256 + hq * 256 + hkv * 2 * (65 + 65 + 128)),
                "flops": rows * ((hq + hkv) * D * 3 + 2 * hkv * D * 3)}
    row = {"f8": 65, "f16": 128, "f32": 256}[c["cache"]]
    P, cap, w = c["prefix"], c["cap"], c["window"]
    # The slots before a sequence's rows are 0 to cap - T, on average half of that.
    filled = (cap - T) / 2
    seen = P + filled + rows / B / 2  # keys of a mean row
    keys = filled + rows / B
    if w:
        seen, keys, P = min(seen, w), min(keys, w + rows / B), min(P, max(0, w))
    return {"bytes": 2 * hkv * row * (P + B * keys) + rows * hq * D * 8, "flops": 4 * D * rows * hq * seen}


# ---------------------------------------------------------------- exact --

def _value64(code, s, width):
    """The values that codes and scale bytes stand for, in 64 bits, from the bits of the format."""
    c = code.to(torch.int64)
    m, e = c & 7, (c >> 3) & 15
    v = torch.where(e > 0, (8 + m).double() * 2.0 ** (e - 10).double(), m.double() * 2.0 ** -9)
    v = torch.where(c > 127, -v, v)
    f = 2.0 ** (s.to(torch.float64) - 127)
    return v * f.repeat_interleave(width, -1)[..., :v.shape[-1]]


def _round64(x, width):
    """x [..., n] rounded to the format in blocks of `width` along the last axis, in 64 bits."""
    n = x.shape[-1]
    b = torch.nn.functional.pad(x.double(), (0, -n % width)).unflatten(-1, (-1, width))
    top = b.abs().amax(-1, keepdim=True)
    e = torch.where(top > 0, torch.ceil(torch.log2(top.clamp_min(1e-300) / 448)), -126.0)
    e = torch.where(448 * 2.0 ** e < top, e + 1, torch.where(448 * 2.0 ** (e - 1) >= top, e - 1, e)).clamp_min(-126.0)
    z = b * 2.0 ** -e
    step = 2.0 ** ((torch.frexp(z.abs())[1] - 1).clamp_min(-6).double() - 3)
    return (torch.round(z / step) * step * 2.0 ** e).flatten(-2)[..., :n]


def exact(case, seed):
    st, c = prepare(case, seed), case
    if c["kind"] == "linear":
        x = _round64(st["x"], 128)
        y = x @ _value64(*st["w"], 128).T
        if c["bias"]:
            y += st["bias"].double()
        if c["gated"]:
            y = y * torch.sigmoid(y) * (x @ _value64(*st["w2"], 128).T)
        if c["gelu"]:
            y = y * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3))
        return y
    B, T, hq, hkv = c["B"], c["T"], c["hq"], c["hkv"]
    pos = st["pos"].tolist()
    n = [T] * B if st["counts"] is None else st["counts"].tolist()
    if c["kind"] == "append":
        q = st["q"].double()
        k, v = st["k16"].double(), st["v16"].double()
        x = st["qkv"].double().view(B, T, hq + 2 * hkv, D)
        for b in range(B):
            p = torch.arange(pos[b], pos[b] + n[b], device="cuda")
            w = torch.outer((p + c["offset"]).double(), st["inv_freq"].double())
            turn = torch.polar(torch.ones_like(w), w)[:, None]
            z = torch.complex(x[b, :n[b], :hq + hkv, :32].contiguous(), x[b, :n[b], :hq + hkv, 32:].contiguous()) * turn
            z = torch.cat([z.real, z.imag], -1)
            q.view(B, T, hq, D)[b, :n[b]] = z[:, :hq]
            k[b, :, p] = _round64(z[:, hq:], D).transpose(0, 1)
            v[b, :, p] = _round64(x[b, :n[b], hq + hkv:], D).transpose(0, 1)
        return {"q": q, "k": k, "v": v}
    val = lambda m, i: (st[m] if i is None else st[m][i])  # noqa: E731
    wide = lambda m, i=None: _value64(val(m, i), val(m + "_scale", i).unsqueeze(-1), D) if c["cache"] == "f8" else val(m, i).double()  # noqa: E731
    P, G = c["prefix"], hq // hkv
    out = st["out"].double()
    pk, pv = (wide("pk")[:, :P], wide("pv")[:, :P]) if P else (None, None)
    for b in range(B):
        ln = pos[b] + n[b]
        k, v = wide("k", b)[:, :ln], wide("v", b)[:, :ln]
        if P:
            k, v = torch.cat([pk, k], 1), torch.cat([pv, v], 1)
        q = st["q"].double().view(B, T, hkv, G, D)[b, :n[b]].permute(1, 2, 0, 3).contiguous()  # [hkv, G, n, 64]
        s = (q @ k.transpose(1, 2)[:, None].contiguous()) * SCALE
        row = torch.arange(P + pos[b], P + ln, device="cuda")[:, None]
        key = torch.arange(P + ln, device="cuda")[None]
        s = s.masked_fill((key > row) | ((key <= row - c["window"]) if c["window"] else (key < 0)), -math.inf)
        o = torch.softmax(s, -1) @ v[:, None]
        out.view(B, T, hkv, G, D)[b, :n[b]] = o.permute(2, 0, 1, 3)
    return out
