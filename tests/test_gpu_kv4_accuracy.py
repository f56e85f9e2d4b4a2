"""Attention over the 4-bit cache against 64 bits by the limits of
kv4_accuracy.py (which test_kv4_accuracy.py shows to tell one f16 number for a
query value or a softmax weight from two)."""
import numpy as np
import pytest

import aspida_amd as aa
import kv4_accuracy as acc
import kv4_plain as plain
from test_gpu_kv4 import NAMES, _attend, _dev, _filled, _host, _starts

pytestmark = pytest.mark.gpu

BITS = {aa.F16: 11, aa.BF16: 8}

# dim, heads, kv, rows, lens, window, in a batch of many rows
CASES = [
    (128, 32, 8, [1] * 8, [3000, 2111, 65, 700, 1000, 33, 512, 1777], 0, False),
    (64, 8, 2, [3, 2, 3], [700, 1300, 90], 0, False),
    (256, 8, 4, [2, 2, 2], [500, 301, 999], 100, False),
    (128, 8, 2, [100, 31], [400, 1500], 0, True),
    (64, 8, 2, [90], [777], 0, True),
    (256, 8, 4, [85], [600], 200, True),
]


@pytest.mark.parametrize("ty", [aa.F32, aa.BF16, aa.F16], ids=NAMES.get)
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"d{c[0]}{'many' if c[6] else 'few'}")
def test_attention_is_as_accurate_as_f32(case, ty):
    dim, heads, kv, rows, lens, window, many = case
    gen = np.random.default_rng(dim + heads + sum(lens))
    c = _filled(gen, dim, kv, lens)
    st, scale = _starts(rows), dim ** -0.5
    q = _dev(2 * gen.standard_normal((st[-1], heads * dim)).astype(np.float32), ty)
    out, lse = _attend(c, ty, q, st, lens, heads, scale, window, many=many)
    ho, hl, hq = _host(out).reshape(-1, heads, dim), _host(lse), _host(q).reshape(-1, heads, dim)
    wo, wl, o32, l32 = [], [], [], []
    for b, (k, v) in enumerate(c.all(lens)):
        rows_of = slice(st[b], st[b + 1])
        o, l, _, _ = plain.attend(hq[rows_of], k, v, scale, window)
        p, m = acc.attend32(hq[rows_of], k, v, scale, window)
        wo.append(o), wl.append(l), o32.append(p), l32.append(m)
    wo, wl, o32, l32 = (np.concatenate(x) for x in (wo, wl, o32, l32))
    assert acc.over(hl, wl, l32) <= 1
    if ty == aa.F32:
        assert acc.over(ho, wo, o32) <= 1
    else:
        assert acc.over16(ho, wo, o32, BITS[ty]) <= 1
