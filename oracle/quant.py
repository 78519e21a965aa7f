"""Groups of values held in few bits, and attention over a cache of them, in 64 bits.

A group keeps lo (its smallest value), step ((largest - smallest) / top rounded to float32) and per
value the code nearest (x - lo) / step; it reads back as lo + code * step.  A group with a value
that is not finite has lo = step = NaN and codes 0.
"""
import numpy as np


def quantise(x, top):
    """codes [..., n] uint32, params [..., 2] float32 of the groups x [..., n] (float32)."""
    x = np.asarray(x, np.float32)
    bad = ~np.isfinite(x).all(-1, keepdims=True)
    x = np.where(bad, np.float32(0), x).astype(np.float64)
    lo, hi = x.min(-1, keepdims=True), x.max(-1, keepdims=True)
    step = ((hi - lo) / float(top)).astype(np.float32)
    with np.errstate(divide="ignore"):
        inv = np.where(step > 0, 1.0 / step.astype(np.float64), 0.0)
    codes = np.minimum(np.rint((x - lo) * inv), top).astype(np.uint32)
    params = np.concatenate([lo.astype(np.float32), step], -1)
    return codes, np.where(bad, np.float32(np.nan), params)


def values(codes, params):
    """What the groups read back as, in 64 bits."""
    p = params.astype(np.float64)
    return p[..., :1] + codes.astype(np.float64) * p[..., 1:]


def pack4(codes):
    """[..., D] -> [..., D/8] uint32, the first code in the lowest bits."""
    c = codes.reshape(*codes.shape[:-1], -1, 8).astype(np.uint32)
    return np.bitwise_or.reduce(c << (4 * np.arange(8, dtype=np.uint32)), axis=-1)


def unpack4(words):
    w = np.asarray(words).astype(np.uint32)
    return ((w[..., None] >> (4 * np.arange(8, dtype=np.uint32))) & 15).reshape(*w.shape[:-1], -1)


def quantise_rows8(x, group=128):
    """codes [rows, round_up(H, 16)] uint8 (padding 0), params [rows, ceil(H/group), 2]."""
    rows, H = x.shape
    codes = np.zeros((rows, (H + 15) // 16 * 16), np.uint8)
    params = []
    for a in range(0, H, group):
        c, p = quantise(x[:, a:a + group], 255)
        codes[:, a:a + c.shape[1]] = c
        params.append(p)
    return codes, np.stack(params, 1)


def values_rows8(codes, params, H, group=128):
    return np.concatenate([values(codes[:, a:min(a + group, H)], params[:, a // group])
                           for a in range(0, H, group)], 1)


def attention(q, k, v, pos, scale, L=None):
    """q [B,T,H,D] over k, v [B,Hk,S,D] (64 bits): query t sees rows j <= pos + t, j < L."""
    B, T, H, D = q.shape
    Hk = k.shape[1]
    L = k.shape[2] if L is None else L
    o = np.empty((B, T, H, D))
    for b in range(B):
        for h in range(H):
            kk, vv = k[b, h // (H // Hk)], v[b, h // (H // Hk)]
            for t in range(T):
                n = min(L, pos + t + 1)
                s = kk[:n] @ q[b, t, h].astype(np.float64) * scale
                p = np.exp(s - s.max())
                o[b, t, h] = p @ vv[:n] / p.sum()
    return o
