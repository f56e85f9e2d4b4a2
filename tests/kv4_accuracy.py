"""Limits for the attention over the 4-bit cache that a lost low half of a
query or of a softmax weight breaks, where the worst-case bounds of
test_gpu_kv4.py do not see it.

They are relative to a plain f32 computation of the same rows (``attend32``,
``weights32``), both measured against 64 bits.  WIDER = 16:
  * 4: a query and a softmax weight are two f16 numbers, which leave 2^-22 of
    a product (the second's half step, 2^-11, of what the first leaves, 2^-11)
    where f32 leaves 2^-24;
  * 4: a key or value is summed as its code's part and its group's minimum.
    For values around 0, d q + m with m about -2 standard deviations and d q
    about 2, the two are together three to four times the value.
f32 results, lse and slot weights: the root mean square of the error, within
WIDER times that of the f32 computation.  16-bit results: an element differs
from the rounded 64-bit one only where that lies as near to a rounding border
as the error before rounding, with a chance of error / step; so the number of
elements that differ has the expectation WIDER sum(|f32 error| / step) at
most, and 5 standard deviations and 5 elements more are allowed.
"""
import numpy as np

import kv4_plain as plain

WIDER = 16


def attend32(q, k, v, scale, window=0):
    """(out, lse) of plain.attend's arguments, every operation in f32."""
    rows, heads, dim = q.shape
    n, kv, _ = k.shape
    q, k, v, f = q.astype(np.float32), k.astype(np.float32), v.astype(np.float32), np.float32(scale)
    out, lse = np.zeros((rows, heads, dim), np.float32), np.full((rows, heads), -np.inf, np.float32)
    see = plain.visible(n, rows, window)
    for h in range(heads):
        g = h * kv // heads
        s = np.where(see, (q[:, h] @ k[:, g].T) * f, np.float32(-np.inf))
        top = s.max(1, keepdims=True)
        p = np.exp(s - top)
        total = p.sum(1, keepdims=True)
        out[:, h] = (p @ v[:, g]) / total
        lse[:, h] = (np.log(total) + top)[:, 0]
    return out, lse


def weights32(q, k, lse, scale, window=0):
    """plain.weights in f32."""
    rows, heads, _ = q.shape
    n, kv, _ = k.shape
    q, k, lse, f = q.astype(np.float32), k.astype(np.float32), lse.astype(np.float32), np.float32(scale)
    acc = np.zeros((kv, n), np.float32)
    see = plain.visible(n, rows, window)
    for h in range(heads):
        g = h * kv // heads
        acc[g] += np.where(see, np.exp((q[:, h] @ k[:, g].T) * f - lse[:, h][:, None]), np.float32(0)).sum(0)
    return acc


def planes(x, n):
    """x as the sum of n f16 numbers."""
    hi = x.astype(np.float16).astype(np.float64)
    return hi if n == 1 else hi + (x - hi).astype(np.float16).astype(np.float64)


def query_planes(q, n):
    """f64 of a query's n f16 numbers, each head's largest value in [2^9, 2^10)."""
    e = np.frexp(np.abs(q).max(-1, keepdims=True))[1]
    return np.ldexp(planes(np.ldexp(q, 10 - e), n), e - 10)


def attend_planes(q, k, v, scale, nq, np_, window=0):
    """(out, lse) in 64 bits but for queries of nq and softmax weights of np_ f16 numbers."""
    q = query_planes(q, nq)
    rows, heads, dim = q.shape
    n, kv, _ = k.shape
    out, lse = np.zeros((rows, heads, dim)), np.zeros((rows, heads))
    see = plain.visible(n, rows, window)
    for h in range(heads):
        g = h * kv // heads
        s = np.where(see, q[:, h] @ k[:, g].T * scale, -np.inf)
        top = s.max(1, keepdims=True)
        p = planes(np.exp(s - top) * 128.0, np_)
        out[:, h] = (p @ v[:, g]) / p.sum(1, keepdims=True)
        lse[:, h] = (np.log(p.sum(1, keepdims=True) / 128.0) + top)[:, 0]
    return out, lse


def rms(x):
    return float(np.sqrt(np.mean(np.square(x)))) if np.size(x) else 0.0


def over(got, want, plain32):
    """The error of f32 results by what is allowed (1: at the limit)."""
    return rms(got - want) / (WIDER * rms(plain32.astype(np.float64) - want))


def round16(x, bits):
    """f64 x at `bits` significant bits (8: bf16, 11: f16), to even; (rounded, step)."""
    e = np.frexp(x)[1] - bits
    step = np.ldexp(1.0, np.maximum(e, -24) if bits == 11 else e)
    return np.rint(x / step) * step, step


def over16(got, want, plain32, bits):
    """How many elements of 16-bit results differ from the rounded 64-bit ones, by what is allowed."""
    r, step = round16(want, bits)
    chance = np.minimum(1.0, WIDER * np.abs(plain32.astype(np.float64) - want) / step).sum()
    return int((got != r).sum()) / (chance + 5 * np.sqrt(chance) + 5)
