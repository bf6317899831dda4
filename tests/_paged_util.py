"""Cases of attention in a window over pages and over contiguous caches, for the tests: inputs on the device, and the
outputs in 64 bits from the definition."""
import numpy as np
import torch

import mingtts as mt
import _f8_util as U

TORCH = {"f32": torch.float32, "f16": torch.float16, "f8": torch.uint8}


def to_pages(x, table, page, pool, fill):
    """Rows x [B, hkv, cap, ...] (numpy) in pages by `table` [B, entries]; the rest of the pool holds `fill`."""
    B, hkv, cap = x.shape[:3]
    out = np.full((pool, hkv, page) + x.shape[3:], fill, x.dtype)
    for b in range(B):
        for e in range(table.shape[1]):
            n = min(page, cap - e * page)
            if n > 0 and 0 <= table[b, e] < pool:
                out[table[b, e], :, :n] = x[b, :, e * page:e * page + n]
    return out


def poison(kind):
    """What unattended slots hold: values and scale bytes that would show."""
    return {"f32": np.float32(np.nan), "f16": np.float16(np.nan), "f8": np.uint8(0x7F)}[kind]


class Case:
    """B sequences of T rows over caches of `cap` slots; page None: contiguous caches.  `hidden` slots, as (b, slot), hold
    NaN and odd scale bytes, as do all that no row attends under (window, sinks)."""

    def __init__(self, gpu, kind, B, T, hq, hkv, cap, page=None, pos=None, counts=None, window=0, sinks=0, seed=0, q_scale=1.0,
                 values=None, missing=()):
        rng = np.random.default_rng(seed + B * 1000 + T * 10 + cap)
        self.gpu, self.kind, self.B, self.T, self.hq, self.hkv, self.cap, self.page = gpu, kind, B, T, hq, hkv, cap, page
        self.window, self.sinks, self.counts, self.missing = window, sinks, counts, set(missing)
        self.pos = [int(rng.integers(0, cap - T + 1)) for _ in range(B)] if pos is None else pos
        self.q = (rng.standard_normal((B * T, hq * 64)) * q_scale).astype(np.float32)
        seen = np.zeros((B, cap), bool)
        for b in range(B):
            for t in range(T if counts is None else counts[b]):
                seen[b, self.keys(b, t)] = True
        self.raw, self.val = [], []
        for i in range(2):
            x = rng.standard_normal((B, hkv, cap, 64)).astype(np.float32)
            if values is not None:
                values(i, x)
            if kind == "f8":
                c, s = U.encode(x, 64)
                self.val.append(U.decode(c, s, 64))
                s = s[..., 0].copy()
            else:
                c, s = x.astype(np.float32 if kind == "f32" else np.float16), None
                self.val.append(c.astype(np.float64))
            hide = ~seen[:, None].repeat(hkv, 1)
            c[hide] = poison(kind)
            if s is not None:
                s[hide] = rng.integers(0, 256, s[hide].shape)
            self.raw.append((c, s))
        d = lambda a: None if a is None else torch.from_numpy(a).to(gpu)  # noqa: E731
        (k, ks), (v, vs) = self.raw
        if page is None:
            self.kv = mt.KV(d(k), d(v), d(ks), d(vs))
            return
        n = (cap + page - 1) // page
        self.pool = B * n + 3
        table = rng.permutation(self.pool)[:B * n].reshape(B, n).astype(np.int32)
        for b, e in self.missing:
            table[b, e] = [-1, self.pool, 2 ** 31 - 1][(b + e) % 3]
        for b in range(B):  # entries of pages that no row sees
            for e in range(n):
                if not seen[b, e * page:(e + 1) * page].any():
                    table[b, e] = -1
        self.table = table
        put = lambda a, fill: None if a is None else d(to_pages(a, table, page, self.pool, fill))  # noqa: E731
        self.kv = mt.PagedKV(put(k, poison(kind)), put(v, poison(kind)), d(table), put(ks, 255), put(vs, 0))

    def keys(self, b, t):
        """The slots that row t of sequence b attends."""
        i = min(self.pos[b] + t, self.cap - 1)
        j = np.arange(i + 1)
        if self.window:
            j = j[(j > i - self.window) | (j < self.sinks)]
        return j[[(b, e // self.page) not in self.missing for e in j]] if self.missing else j

    def run(self, len_max=0, scale=0.125, stream=None, workspace=None, pad=0, kv=None):
        i = lambda a: None if a is None else torch.tensor(a, dtype=torch.int32, device=self.gpu)  # noqa: E731
        n = self.B * self.T
        q = torch.zeros(n, self.hq * 64 + pad, device=self.gpu)
        q[:, :self.hq * 64] = torch.from_numpy(self.q).to(self.gpu)
        out = torch.full((n + 1, self.hq * 64 + pad), -5.0, device=self.gpu)
        call = mt.attention_sinks if self.page is None else mt.attention_paged
        pos, counts = i(self.pos), i(self.counts)
        torch.cuda.synchronize()
        call(q, self.B, self.T, self.hq, self.hkv, pos, kv or self.kv, out, window=self.window, sinks=self.sinks, counts=counts,
             len_max=len_max, scale=scale, stream=stream, workspace=workspace)
        torch.cuda.synchronize()
        out = out.cpu().double().numpy()
        assert (out[-1] == -5).all() and (out[:, self.hq * 64:] == -5).all()
        return out[:-1, :self.hq * 64].reshape(self.B, self.T, self.hq, 64)

    def want(self, b, t, h, scale=0.125):
        kh, j = h // (self.hq // self.hkv), self.keys(b, t)
        if len(j) == 0:
            return np.zeros(64), 0.0
        k, v = (x[b, kh, j] for x in self.val)
        return U.attend64(self.q.reshape(self.B, self.T, self.hq, 64)[b, t, h].astype(np.float64), k, v, 0, len(j), scale)

    def check(self, got, scale=0.125, rows=None):
        err = norm = 0.0
        for b in range(self.B):
            for t in range(self.T):
                if t >= (self.T if self.counts is None else self.counts[b]):
                    assert (got[b, t] == -5).all()
                    continue
                if rows is not None and (b, t) not in rows:
                    continue
                for h in range(self.hq):
                    want, tol = self.want(b, t, h, scale)
                    worst = np.abs(got[b, t, h] - want).max()
                    assert worst <= tol, f"row {b} {t} head {h}: off by {worst:.3g}, bound {tol:.3g}"
                    err += ((got[b, t, h] - want) ** 2).sum()
                    norm += (want ** 2).sum()
        rel = np.sqrt(err / norm) if norm else 0.0
        assert rel <= 5e-6, rel
        return rel
