"""Plain 64-bit forms of the rotary and 4-bit cache calls (numpy, no layout):
what the tests of test_kv4.py and test_gpu_kv4.py compare with."""
import math

import numpy as np


def rope_freqs(rot, base, scaling="none", factor=1.0, low=1.0, high=4.0, context=0, freq_factors=None):
    i = np.arange(rot // 2, dtype=np.float64)
    f = base ** (-2.0 * i / rot)
    if freq_factors is not None:
        f = f / np.asarray(freq_factors, np.float32).astype(np.float64)
    if scaling == "linear":
        return f / factor
    if scaling == "bands":
        s = np.clip((context * f / (2 * np.pi) - low) / (high - low), 0, 1)
        return (1 - s) * f / factor + s * f
    if scaling == "yarn":
        def at(t):
            return rot * math.log(context / (t * 2 * math.pi)) / (2 * math.log(base))
        lo, hi = max(math.floor(at(high)), 0), min(math.ceil(at(low)), rot - 1)
        r = np.clip((i - lo) / max(hi - lo, 0.001), 0, 1)
        return f / factor * r + f * (1 - r)
    return f


def rotate(x, pos, freqs, mag, interleaved, inverse=False):
    """f64 x [tokens][heads][dim] rotated."""
    x = np.asarray(x, np.float64)
    y, half = x.copy(), len(freqs)
    a = np.asarray(pos, np.float64)[:, None] * freqs
    c, s = np.cos(a)[:, None] * mag, np.sin(a)[:, None] * mag * (-1 if inverse else 1)
    p = np.arange(half)
    u, w = (2 * p, 2 * p + 1) if interleaved else (p, p + half)
    y[..., u] = x[..., u] * c - x[..., w] * s
    y[..., w] = x[..., u] * s + x[..., w] * c
    return y


def quantise(x):
    """(d, m, q) of f32 x [..., dim]: shapes [..., groups], [..., groups], [..., groups, 32]."""
    x = np.asarray(x, np.float32)
    g = x.reshape(*x.shape[:-1], -1, 32).astype(np.float64)
    with np.errstate(all="ignore"):
        m = g.min(-1).astype(np.float32).astype(np.float16).astype(np.float64)
        r = (g.max(-1) - m) / 15.0
        e = np.frexp(np.where(np.isfinite(r) & (r > 0), r, 1.0))[1]
        step = np.exp2(np.maximum(e - 7, -24).astype(np.float64))
        d = np.where(r > 0, np.ceil(r / step) * step, 0.0)
        bad = ~np.isfinite(g).all(-1) | ~np.isfinite(m) | (d > 254)
        q = np.where(d[..., None] > 0, np.rint((g - m[..., None]) / np.where(d > 0, d, 1)[..., None]), 0)
        q = np.clip(q, 0, 15)
    return np.where(bad, np.nan, d), np.where(bad, 0, m), np.where(bad[..., None], 0, q)


def stands_for(x):
    """f64 values that the cache holds for f32 x [..., dim]."""
    d, m, q = quantise(x)
    return (q * d[..., None] + m[..., None]).reshape(np.shape(x))


def pair_stands_for(k, v):
    """The same for the keys and values of the same tokens and heads: where
    either has a group beyond the format, both are NaN."""
    k, v = stands_for(k), stands_for(v)
    bad = np.isnan(k).any(-1) | np.isnan(v).any(-1)
    k[bad] = v[bad] = np.nan
    return k, v


def visible(n, rows, window):
    """bool [rows][n]: which slots each of the last `rows` of n tokens sees."""
    pos = np.arange(n - rows, n)[:, None]
    j = np.arange(n)[None, :]
    see = j <= pos
    if window > 0:
        see &= j > pos - window
    return see


def parts(x):
    """|d q| + |m| at least, of cached values x [..., dim]: a value is the sum
    of its code's part and its group's minimum (code 0 occurs in each group)."""
    m = x.reshape(*x.shape[:-1], -1, 32).min(-1)
    return np.abs(x) + 2 * np.repeat(np.abs(m), 32, -1)


def attend(q, k, v, scale, window=0):
    """q [rows][heads][dim], k and v [n][kv][dim] f64 -> (out, lse, sum p parts(v),
    largest visible scale * sum |q| parts(k)) of the rows at the end of the n
    slots."""
    rows, heads, dim = q.shape
    n, kv, _ = k.shape
    out = np.zeros((rows, heads, dim))
    lse = np.full((rows, heads), -np.inf)
    pv, sk = np.zeros((rows, heads, dim)), np.zeros((rows, heads))
    see = visible(n, rows, window)
    kp, vp = parts(k), parts(v)
    for h in range(heads):
        g = h * kv // heads
        with np.errstate(invalid="ignore"):
            s = q[:, h] @ k[:, g].T * scale
            size = np.abs(q[:, h]) @ kp[:, g].T * abs(scale)
        for r in range(rows):
            w = see[r]
            if not w.any():
                continue
            top = s[r, w].max()
            p = np.exp(s[r, w] - top)
            lse[r, h] = top + np.log(p.sum())
            p /= p.sum()
            out[r, h] = p @ v[w, g]
            pv[r, h] = p @ vp[w, g]
            sk[r, h] = size[r, w].max()
    return out, lse, pv, sk


def weights(q, k, lse, scale, window=0):
    """f64 [kv][n]: the weight each slot receives."""
    rows, heads, _ = q.shape
    n, kv, _ = k.shape
    acc = np.zeros((kv, n))
    see = visible(n, rows, window)
    for h in range(heads):
        g = h * kv // heads
        s = q[:, h] @ k[:, g].T * scale
        with np.errstate(invalid="ignore", over="ignore"):
            p = np.where(see & np.isfinite(lse[:, h])[:, None], np.exp(s - lse[:, h][:, None]), 0.0)
        acc[g] += p.sum(0)
    return acc


def keep_slots(acc, n, keep, first, recent):
    """Kept slots, ascending, by one head's weights."""
    if n <= keep:
        return np.arange(n)
    w = np.zeros(n)
    m = min(n, len(acc))
    a = np.asarray(acc[:m], np.float64)
    w[:m] = np.where(a > 0, a, 0.0)
    mid = np.arange(first, n - recent)
    order = mid[np.argsort(-w[mid], kind="stable")][:keep - first - recent]
    return np.sort(np.concatenate([np.arange(first), order, np.arange(n - recent, n)])).astype(np.int64)
