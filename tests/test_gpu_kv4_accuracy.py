"""Attention over the 4-bit cache against 64 bits by the limits of
kv4_accuracy.py (which test_kv4_accuracy.py shows to tell one f16 number for a
query value or a softmax weight from two)."""
import numpy as np
import pytest

import aspida_amd as aa
import kv4_accuracy as acc
import kv4_plain as plain
from gpu_helpers import stream, sync, torch_cuda
from test_gpu_kv4 import NAMES, Cache, _attend, _check, _dev, _filled, _host, _i32, _kv, _starts

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


@pytest.mark.parametrize("rows,many", [(3, False), (90, True)], ids=["few", "many"])
@pytest.mark.parametrize("ty", [aa.F32, aa.BF16], ids=NAMES.get)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_attention_of_values_at_the_ends_of_f16(dim, ty, rows, many):
    """Groups whose minimum, and whose minimum and half its range, lie at f16's
    largest values or beyond them, in sight of some of the rows."""
    gen = np.random.default_rng(dim)
    heads, kv, n = 8, 2, 150
    k, v = _kv(gen, n, kv, dim)
    g = v.reshape(n, kv, dim // 32, 32)
    codes = np.concatenate([np.arange(16), np.arange(16)]).astype(np.float32)
    g[n - 20, :, 1] = 64000 + 250 * gen.permutation(codes)
    g[n - 50, 0, 0] = -65504 + 254 * gen.permutation(codes)
    g[n - 1, 1, 0] = 65504 + 254 * gen.permutation(codes)
    c = Cache(gen, dim, kv, 1, 3)
    c.append(aa.F32, _dev(k), _dev(v), [0, n], [n])
    kvs = c.all([n])
    assert np.isfinite(kvs[0][1]).all() and kvs[0][1].max() == 65504 + 15 * 254
    q, scale = _dev(2 * gen.standard_normal((rows, heads * dim)).astype(np.float32), ty), dim ** -0.5
    out, lse = _attend(c, ty, q, [0, rows], [n], heads, scale, many=many)
    _check(c, ty, q, [0, rows], [n], heads, scale, 0, out, lse, kvs)
    if ty == aa.F32:
        hq = _host(q).reshape(rows, heads, dim)
        want = plain.attend(hq, *kvs[0], scale)[0]
        assert acc.over(_host(out).reshape(want.shape), want, acc.attend32(hq, *kvs[0], scale)[0]) <= 1


@pytest.mark.parametrize("ty", [aa.F32, aa.BF16, aa.F16], ids=NAMES.get)
@pytest.mark.parametrize("scale", [1.0, -1.0], ids=["plus", "minus"])
@pytest.mark.parametrize("case", [
    (128, 32, 8, [1] * 6, [3000, 65, 700, 1000, 33, 512], 0),
    (64, 8, 2, [3, 2, 3], [700, 1300, 90], 0),
    (256, 8, 4, [2, 2], [500, 301], 100),
    (128, 8, 2, [40, 31], [400, 900], 0),
    (64, 8, 2, [90], [777], 0),
    (256, 8, 4, [20, 1], [600, 70], 200),
], ids=lambda c: f"d{c[0]}r{c[3][0]}")
def test_slot_weights_are_as_accurate_as_f32(case, scale, ty):
    """Each slot's weight, for negative scales and query rows at an odd stride too."""
    dim, heads, kv, rows, lens, window = case
    torch = torch_cuda()
    gen = np.random.default_rng(dim + heads + sum(lens))
    c = _filled(gen, dim, kv, lens)
    st, scale = _starts(rows), scale * dim ** -0.5
    wide = heads * dim + 3
    q = _dev(2 * gen.standard_normal((st[-1], wide)).astype(np.float32), ty)
    _, lse = _attend(c, ty, q, st, lens, heads, scale, window)
    stride = max(lens)
    out = torch.full((len(lens), kv, stride), 7.0, device="cuda")
    s, l = _i32(st), _i32(lens)
    c.dev.kv4_weigh(c.c, ty, q.data_ptr(), wide, heads, int(st[-1]), len(lens), s.data_ptr(), max(rows), l.data_ptr(),
                    scale, lse.data_ptr(), 0, out.data_ptr(), stride, stream(), window=window)
    sync()
    got, hl, hq = _host(out), _host(lse), _host(q)[:, :heads * dim].reshape(-1, heads, dim)
    ratio, ratio32 = [], []
    for b, (k, v) in enumerate(c.all(lens)):
        r, n = slice(st[b], st[b + 1]), lens[b]
        want = plain.weights(hq[r], k, hl[r], scale, window)
        w32 = acc.weights32(hq[r], k, hl[r], scale, window)
        assert (got[b][:, n:] == 0).all() and (got[b][:, :n][want == 0] == 0).all()
        some = want > 1e-30
        ratio.append(got[b][:, :n][some] / want[some])
        ratio32.append(w32[some] / want[some])
    assert acc.over(np.concatenate(ratio), 1.0, np.concatenate(ratio32)) <= 1
