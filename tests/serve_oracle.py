"""The serving operators in plain numpy, in 64 bits, from their definitions: one sequence, one page, one row at a time."""
import math

import numpy as np

E4M3_MAX = 448.0


def e4m3_value(codes):
    """float64 values of e4m3 codes (uint8)."""
    c = codes.astype(np.int64)
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))
    return np.where(c & 128, -v, v)


def prepared(x, w, pos, rope, theta, eps, freq=None, norm=True):
    """x[heads, hd] normed (w may be None for a norm without weight; norm=False: none) and rotated to `pos`."""
    x = x.astype(np.float64)
    hd = x.shape[-1]
    if norm:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
        x = x if w is None else x * w.astype(np.float64)
    if rope == 0:
        return x
    j = np.arange(hd // 2)
    a = pos * theta ** (-2.0 * j / hd) / (1.0 if freq is None else freq.astype(np.float64))
    i0, i1 = (j, j + hd // 2) if rope == 1 else (2 * j, 2 * j + 1)
    y = x.copy()
    y[..., i0] = x[..., i0] * np.cos(a) - x[..., i1] * np.sin(a)
    y[..., i1] = x[..., i0] * np.sin(a) + x[..., i1] * np.cos(a)
    return y


def scale_for(amax):
    """The least power of two s >= 2^-120 with amax <= 448 s."""
    s = 2.0 ** -120
    if amax > 0:
        s = max(s, 2.0 ** (math.frexp(amax / E4M3_MAX)[1] - 1))
        if amax > E4M3_MAX * s:
            s *= 2.0
    return s


def attend(q, k, v, last, scale, window=0, hole=None):
    """q[heads, hd] against k, v[tokens, n_kv, hd]; sees tokens last - window + 1 .. last that are cached and not in `hole`."""
    heads, hd = q.shape
    n_kv = k.shape[1]
    out = np.zeros((heads, hd))
    t = np.arange(k.shape[0])
    see = (t <= last) & ((t > last - window) if window else True)
    if hole is not None:
        see &= ~hole
    if not see.any():
        return out
    for h in range(heads):
        kv = h // (heads // n_kv)
        s = (k[see, kv].astype(np.float64) @ q[h].astype(np.float64)) * scale
        p = np.exp(s - s.max())
        out[h] = p @ v[see, kv].astype(np.float64) / p.sum()
    return out


def draw(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(id, probability) of one row of logits, in float64."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    m = x.max()
    if m == -np.inf:
        return 0, 0.0
    order = np.argsort(-x, kind="stable")
    if not temperature > 0:
        return int(order[0]), 1.0
    if 0 < top_k < len(x):
        order = order[:top_k]
    with np.errstate(invalid="ignore"):
        w = np.where(x[order] == m, 1.0, 0.0 if m == np.inf else np.exp((x[order] - m) / temperature))
    if top_p < 1:
        before = np.cumsum(w) - w
        keep = before < top_p * w.sum()
        keep[0] = True
        order, w = order[keep], w[keep]
    keep = (w >= min_p) | (x[order] == m)
    order, w = order[keep], w[keep]
    by = np.argsort(order)
    order, w = order[by], w[by]
    c = np.cumsum(w)
    i = min(int(np.searchsorted(c, u * c[-1], side="right")), len(w) - 1)
    return int(order[i]), float(w[i] / c[-1])
