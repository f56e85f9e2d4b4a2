"""Plain 64-bit forms of trees of drafted tokens and of products with 8-bit
integer weights (numpy, no layout)."""
import math

import numpy as np

import kv4_plain as plain


# ---- trees -------------------------------------------------------------------

def tree_parent(parent, i):
    p = int(parent[i])
    return p if 0 <= p < i else -1


def ancestors(parent):
    """bool [n][n]: row i's ancestors and itself."""
    n = len(parent)
    on = np.zeros((n, n), bool)
    for i in range(n):
        p = tree_parent(parent, i)
        if p >= 0:
            on[i] = on[p]
        on[i, i] = True
    return on


def mask_words(on, words):
    """uint32 [n][words] of bool [n][m]; columns past 32 * words are left out."""
    n, m = on.shape
    bits = np.zeros((n, 32 * words), bool)
    bits[:, :min(m, 32 * words)] = on[:, :32 * words]
    return (bits.reshape(n, words, 32).astype(np.uint64) << np.arange(32, dtype=np.uint64)).sum(-1).astype(np.uint32)


def tree_sees(on, base, window):
    """bool [n][base + n] (base may be negative: slots from 0 on) of rows whose
    mask is bool [n][n]."""
    n = len(on)
    see = np.zeros((n, max(base + n, 0)), bool)
    for i in range(n):
        if base + i < 0:
            continue
        rows = [j for j in range(n) if on[i, j] and base + j >= 0]
        low = max(0, base - max(window - len(rows), 0)) if window else 0
        see[i, low:max(base, 0)] = True
        see[i, [base + j for j in rows]] = True
    return see


def attend(q, k, v, scale, see):
    """As kv4_plain.attend, with bool see [rows][n]."""
    rows, heads, dim = q.shape
    kv = k.shape[1]
    out = np.zeros((rows, heads, dim))
    lse = np.full((rows, heads), -np.inf)
    pv, sk = np.zeros((rows, heads, dim)), np.zeros((rows, heads))
    if not len(k):
        return out, lse, pv, sk
    kp, vp = plain.parts(k), plain.parts(v)
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


def says(row):
    """The token of the largest logit, -1 where all are NaN."""
    row = np.asarray(row, np.float64)
    if np.isnan(row).all():
        return -1
    return int(np.argmax(np.where(np.isnan(row), -np.inf, row) == np.nanmax(row)))


def accept(logits, parent, token):
    """(path, next) of one sequence."""
    n = len(parent)
    if n == 0:
        return [], -1
    path = [0]
    while True:
        said = says(logits[path[-1]])
        child = [i for i in range(path[-1] + 1, n)
                 if tree_parent(parent, i) == path[-1] and token[i] == said and said >= 0]
        if not child:
            return path, said
        path.append(child[0])


# ---- 8-bit numbers -------------------------------------------------------------

def quantise8(x):
    """(f64 scales that are f32 numbers, f64 codes) of the rows of f32 x."""
    x = np.asarray(x, np.float32).astype(np.float64)
    with np.errstate(invalid="ignore"):
        top = np.abs(x).max(-1)
        s = (top / 127).astype(np.float32).astype(np.float64)
        s = np.where(np.isfinite(x).all(-1), np.where(top < 2.0 ** -100, 0.0, s), np.nan)
        live = np.isfinite(s) & (s > 0)
        c = np.where(live[..., None], np.rint(x / np.where(live, s, 1.0)[..., None]), 0.0)
    return s, c


def product8(x, codes, scale):
    """f64 [rows][out] of f32 x, integer codes [out][in] and f32 scales [out]."""
    s, c = quantise8(x)
    with np.errstate(invalid="ignore"):
        return (c @ np.asarray(codes, np.float64).T) * s[:, None] * np.asarray(scale, np.float64)


def gate_argument(g, act):
    return g if act == 0 else 2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)


def activation(g, act):
    """silu, or gelu in its tanh form."""
    with np.errstate(over="ignore", invalid="ignore"):
        return g / (1 + np.exp(-gate_argument(g, act)))
