"""Plain restatements in 64 bits of the 4-bit cache format and of attention
with shaped scores (include/lt_kv.h), for the tests of their kernels."""
from __future__ import annotations

import numpy as np

GROUP, MAX_SCALE = 32, 2720.0


def round_sig(a: np.ndarray, bits: int) -> np.ndarray:
    """a >= 0 rounded to `bits` significant bits, ties to even."""
    m, e = np.frexp(np.asarray(a, np.float64))
    return np.ldexp(np.round(m * 2.0 ** bits), e - bits)


def quant4(x: np.ndarray):
    """x [..., D] -> codes [..., D] in 0..15 and signed scales [..., D/32] f64."""
    g = np.asarray(x, np.float64).reshape(*x.shape[:-1], -1, GROUP)
    mag = np.where(np.isnan(g), 0.0, np.abs(g))
    top = mag.max(-1, keepdims=True)
    a = np.where(np.isinf(top), MAX_SCALE, np.minimum(round_sig(np.where(np.isinf(top), 0, top) / 8, 8), MAX_SCALE))
    a = a.astype(np.float16).astype(np.float64)
    positive = ((g == top) & (top > 0)).any(-1, keepdims=True) | (top == 0)
    d = np.where(positive, -a, a)
    with np.errstate(invalid="ignore", divide="ignore"):
        c = np.floor(g / d + 0.5) + 8
    c = np.where((a == 0) | np.isnan(g), 8, np.clip(c, 0, 15))
    return c.reshape(x.shape).astype(np.uint8), d[..., 0]


def value4(codes: np.ndarray, d: np.ndarray) -> np.ndarray:
    return (codes.astype(np.float64) - 8) * np.repeat(d, GROUP, -1)


def quant8(x: np.ndarray):
    """Q8_0 values q * d of x in 64 bits (LT_KV_Q8_0, f32 arithmetic for d and q)."""
    g = np.asarray(x, np.float32).reshape(*x.shape[:-1], -1, GROUP)
    d = (np.abs(g).max(-1, keepdims=True) / np.float32(127)).astype(np.float32)
    with np.errstate(divide="ignore", invalid="ignore"):
        inv = np.where(d > 0, np.float32(1) / d, np.float32(0))
    y = (g * inv).astype(np.float32)
    q = np.clip(np.trunc(y + np.copysign(np.float32(0.5), y)), -128, 127)
    return (q.astype(np.float64) * d.astype(np.float16).astype(np.float64)).reshape(x.shape)


def attend(q, k, v, pos, group, scale, *, softcap=0.0, window=0, slopes=None, first=None, end=None):
    """One token: q [Hq, D]; k, v [L, Hkv, D] -> [Hq, D] f64.  Masked cells are
    left out before anything is computed from them."""
    lo, hi = (0 if first is None else int(first)), (pos + 1 if end is None else int(end))
    if window:
        lo = max(lo, pos + 1 - window)
    out = np.zeros(q.shape, np.float64)
    if lo >= hi:
        return out
    j = np.arange(lo, hi)
    for h in range(q.shape[0]):
        s = scale * (k[lo:hi, h // group].astype(np.float64) @ q[h].astype(np.float64))
        if softcap:
            s = softcap * np.tanh(s / softcap)
        if slopes is not None:
            s = s - np.float64(slopes[h]) * np.abs(pos - j)
        w = np.exp(s - s.max())
        out[h] = (w / w.sum()) @ v[lo:hi, h // group].astype(np.float64)
    return out
