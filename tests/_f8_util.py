"""The 8-bit format and its operators in 64 bits, for the tests: plain numpy / torch on the CPU."""
import math

import numpy as np
import torch

EPS32 = 2.0 ** -24  # half a step of fp32


def table() -> np.ndarray:
    """The values of the 256 codes."""
    v = np.empty(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        x = math.nan if c & 127 == 127 else (8 + m) * 2.0 ** (e - 10) if e else m * 2.0 ** -9
        v[c] = -x if c > 127 else x
    return v


TABLE = table()


def decode(codes, scales, width):
    """Values of codes [..., n] with scale bytes [..., blocks] (more are ignored), float64."""
    c = np.asarray(codes, np.uint8)
    f = np.repeat(2.0 ** (np.asarray(scales, np.float64) - 127), width, -1)[..., :c.shape[-1]]
    return TABLE[c] * f


def encode(x, width):
    """Codes and scale bytes of x [..., n] by the definition: a search for the scale, then the nearest code
    (ties to the even one) of each value."""
    x = np.asarray(x, np.float64)
    n = x.shape[-1]
    pad = np.zeros(x.shape[:-1] + (-n % width,))
    b = np.concatenate([x, pad], -1).reshape(*x.shape[:-1], -1, width)
    top = np.where(np.isfinite(b), np.abs(b), 0).max(-1)
    s = np.ones(top.shape, int)
    for e in range(-126, 122):
        s = np.where(top > 448 * 2.0 ** e, e + 1 + 127, s)
    z = np.abs(b * 2.0 ** (127.0 - s)[..., None])
    pos = TABLE[:127]
    i = np.clip(np.searchsorted(pos, np.where(np.isfinite(z), z, 0)), 1, 126)
    lo, hi = pos[i - 1], pos[i]
    up = (z - lo > hi - z) | ((z - lo == hi - z) & (i % 2 == 0))
    code = np.where(up, i, i - 1)
    code = np.where(np.isfinite(b), code, 127).astype(np.uint8) | np.where(np.signbit(b), 128, 0).astype(np.uint8)
    return code.reshape(*x.shape[:-1], -1)[..., :n], s.astype(np.uint8)


def rope64(x, position, inv_freq):
    """NeoX rotation of heads x [..., 64] at `position`, 64 bits from the fp32 frequencies."""
    a = float(position) * np.asarray(inv_freq, np.float64)
    c, s = np.cos(a), np.sin(a)
    lo, hi = x[..., :32], x[..., 32:]
    return np.concatenate([lo * c - hi * s, hi * c + lo * s], -1)


def attend64(q, k, v, lo, hi, scale):
    """One query head q [64] over rows lo .. hi - 1 of k, v [n, 64]; also the bound of an fp32 kernel's error.

    Scores: a dot of 64 rounded products and sums is off by 67 half steps of sum |q k|; an error d of a score
    moves a weight by d and the fraction by at most 2 d of the largest |v|.  The sums over keys are
    taken 32 at a time and joined: 64 + n / 32 roundings above and below the fraction; the exponential and the
    division add 8."""
    s = (k[lo:hi] @ q) * scale
    p = np.exp(s - s.max())
    out = (p[:, None] * v[lo:hi]).sum(0) / p.sum()
    d = 67 * EPS32 * abs(scale) * (np.abs(k[lo:hi]) @ np.abs(q)).max()
    tol = np.abs(v[lo:hi]).max() * (2 * d + (2 * (64 + (hi - lo) / 32) + 8) * EPS32)
    return out, tol


def cache(shape, kind, rng, device):
    """A cache's torch tensor(s) of N(0, 1) values of type f32, f16 or f8, and the values in 64 bits."""
    x = rng.standard_normal(shape + (64,)).astype(np.float32)
    if kind == "f32":
        return torch.from_numpy(x).to(device), None, x.astype(np.float64)
    if kind == "f16":
        h = x.astype(np.float16)
        return torch.from_numpy(h).to(device), None, h.astype(np.float64)
    c, s = encode(x, 64)
    return (torch.from_numpy(c).to(device), torch.from_numpy(s[..., 0].copy()).to(device), decode(c, s, 64))
