"""Rotary positions and the 4-bit cache on the GPU against plain 64-bit forms.

Bounds, with u = 2^-24 (half a step of f32) and h_T half a step of the type:
  * a result of the type rounds by h_T of itself, or half its subnormals' spacing;
  * rope: each product and the table's cos and sin round once in f32:
    4 u mag (|a| + |b|), plus h_T of the result;
  * append and read: the stored value exactly, rounded to f32 and the type;
  * scores: the two f16 planes of a query leave 2^-22 of each product, and the
    f32 sums at most 16 roundings of partial sums: S = 2^-19 of
    scale sum |q| (|d code| + |m|), a key being summed as its code's part and
    its minimum apart;
  * attention: a softmax weight is off by the two scores' errors, 2 S, exp
    (2^-22) and its own planes (2^-22), the sums by a rounding per addition
    of a lane (n / 16 + 64 of them at most): E_w = 2 S + 2^-20 +
    (n / 16 + 64) u.  With f16 and bf16 activations weights and values are
    single f16 numbers: 2^-11 more each.  The output: E_w sum p (|d code| + |m|), plus h_T;
  * lse: S + 2^-20 + (n / 16 + 64) u + u |lse|;
  * weights of slots: each term S + u |score - lse| scale + 2^-20, all
    positive: summed.
"""
import numpy as np
import pytest

import aspida_amd as aa
import kv4_plain as plain
from gpu_helpers import stream, sync, torch_cuda

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {aa.F32: 2.0 ** -24, aa.F16: 2.0 ** -11, aa.BF16: 2.0 ** -8}
# Half the spacing of a type's subnormals: f16's is 2^-24 below 2^-14.
TINY = {aa.F32: 2.0 ** -126, aa.F16: 2.0 ** -25, aa.BF16: 2.0 ** -126}
NAMES = {aa.F32: "f32", aa.F16: "f16", aa.BF16: "bf16"}


def _t(ty):
    torch = torch_cuda()
    return {aa.F32: torch.float32, aa.F16: torch.float16, aa.BF16: torch.bfloat16}[ty]


def _dev(a, ty=None):
    t = torch_cuda().from_numpy(np.ascontiguousarray(a)).cuda()
    return t if ty is None else t.to(_t(ty))


def _host(t):
    return t.detach().float().cpu().numpy().astype(np.float64)


def _i32(v):
    return _dev(np.asarray(v, np.int32))


# ---- rope --------------------------------------------------------------------

ROPES = [
    # type, tokens, heads, dim, rot, interleaved, first position, spare elements per row
    (aa.F32, 1, 40, 128, 128, False, 1000, 0),
    (aa.F32, 1, 1, 2, 2, True, 0, 0),
    (aa.F32, 7, 3, 80, 20, False, 12345, 3),      # runs of 10 and 60: pairs
    (aa.F32, 5, 2, 9, 6, False, 77, 1),           # runs of 3: single values
    (aa.BF16, 133, 9, 128, 64, True, 400000, 0),
    (aa.F16, 65, 5, 256, 256, False, 1000000, 8),
    (aa.F16, 3, 2, 64, 64, True, -5, 5),          # rows that start at odd elements
    (aa.BF16, 300, 72, 128, 128, False, 2000, 0),
    (aa.F32, 2000, 3, 96, 32, True, 0, 0),
]


@pytest.mark.parametrize("case", ROPES, ids=lambda c: f"{NAMES[c[0]]}t{c[1]}h{c[2]}d{c[3]}r{c[4]}{'i' if c[5] else 'h'}")
@pytest.mark.parametrize("place", ["apart", "in_place"])
def test_rope(case, place):
    ty, n, heads, dim, rot, inter, p0, spare = case
    torch = torch_cuda()
    gen = np.random.default_rng(n + heads + dim)
    kw = dict(scaling="yarn", factor=4.0, low=1.0, high=32.0, context=8192) if rot > 8 else {}
    rope = aa.Rope(rot, base=10000.0, layout="interleaved" if inter else "half", **kw)
    f, mag = rope.table()
    stride = heads * dim + spare
    buf = _dev(gen.standard_normal((n, stride)).astype(np.float32), ty)
    before = _host(buf)
    x = before[:, :heads * dim].reshape(n, heads, dim)
    pos = p0 + np.arange(n) * (1 if n > 10 else -3)
    out = buf if place == "in_place" else torch.full((n, stride), 7.0, dtype=_t(ty), device="cuda")
    fill = before if place == "in_place" else np.full((n, stride), 7.0)
    dp = _i32(pos)
    for inverse in ((False,) if place == "in_place" else (False, True)):
        aa.DeviceOps().rope(rope, ty, buf.data_ptr(), stride, n, heads, dim, dp.data_ptr(), out.data_ptr(), stride,
                            stream(), inverse=inverse)
        sync()
        got = _host(out)
        want = plain.rotate(x, pos, f, mag, inter, inverse)
        i = np.arange(rot // 2)
        u, w = (2 * i, 2 * i + 1) if inter else (i, i + rot // 2)
        size = np.zeros_like(want)
        size[..., u] = size[..., w] = np.abs(x[..., u]) + np.abs(x[..., w])
        bound = 4 * U * mag * size + HALF[ty] * np.abs(want) * (1 + 2.0 ** -10) + TINY[ty]
        err = np.abs(got[:, :heads * dim].reshape(want.shape) - want)
        assert np.all(err <= bound), np.max(err / bound)
        assert np.array_equal(got[:, :heads * dim].reshape(want.shape)[..., rot:], x[..., rot:])
        assert np.array_equal(got[:, heads * dim:], fill[:, heads * dim:])


def test_rope_inverse_is_the_gradient_and_undoes_it():
    """Against differences of sum(w * rope(x)) in f64, and back to x."""
    torch = torch_cuda()
    gen = np.random.default_rng(5)
    rope = aa.Rope(16, base=100.0)
    x, w, pos = gen.standard_normal((6, 2, 20)), gen.standard_normal((6, 2, 20)), np.arange(6) * 1000
    g = _dev(w.astype(np.float32))
    out = torch.empty_like(g)
    dp = _i32(pos)
    dev = aa.DeviceOps()
    dev.rope(rope, aa.F32, g.data_ptr(), 40, 6, 2, 20, dp.data_ptr(), out.data_ptr(), 40, stream(), inverse=True)
    f, mag = rope.table()
    num = np.zeros_like(x)
    eps = 1e-4
    for i in np.ndindex(x.shape):
        e = np.zeros_like(x)
        e[i] = eps
        num[i] = ((plain.rotate(x + e, pos, f, mag, False) - plain.rotate(x - e, pos, f, mag, False)) * w).sum() / (2 * eps)
    # The map is linear: differences are exact up to f64 rounding / eps, about 1e-10.
    assert np.all(np.abs(_host(out) - num) <= 4 * U * 2 * np.abs(w).max() + 1e-9)
    dev.rope(rope, aa.F32, out.data_ptr(), 40, 6, 2, 20, dp.data_ptr(), out.data_ptr(), 40, stream())
    sync()
    assert np.all(np.abs(_host(out) - w.astype(np.float32)) <= 16 * U * np.abs(w).max())


# ---- the cache ---------------------------------------------------------------

class Cache:
    """A pool with its pages in random order, filled with 0xFF bytes (NaN
    scales) so that whatever is read without having been written shows."""

    def __init__(self, gen, dim, kv, n_seq, max_pages, spare=3, fill=0xFF):
        torch = torch_cuda()
        self.dev = aa.DeviceOps()
        self.dim, self.kv, self.n_seq, self.max_pages = dim, kv, n_seq, max_pages
        self.pool = n_seq * max_pages + spare
        self.pages = torch.full((self.pool, kv * 80 * dim), fill, dtype=torch.uint8, device="cuda")
        self.host_table = gen.permutation(self.pool)[:n_seq * max_pages].astype(np.int32).reshape(n_seq, max_pages)
        self.set_table(self.host_table)

    def set_table(self, t):
        self.table = _i32(t)
        self.c = aa.KV4Cache(self.dim, self.kv, self.pool, self.max_pages, self.pages.data_ptr(), self.table.data_ptr())

    def append(self, ty, k, v, starts, lens, rope=None, pos=None, stride=None):
        n = k.shape[0]
        self.keep = (_i32(starts) if starts is not None else None, _i32(lens), None if pos is None else _i32(pos))
        self.dev.kv4_append(self.c, ty, k.data_ptr(), stride or self.kv * self.dim, v.data_ptr(),
                            stride or self.kv * self.dim, n, len(lens), self.keep[0].data_ptr() if starts is not None else 0,
                            self.keep[1].data_ptr(), rope, 0 if pos is None else self.keep[2].data_ptr(), stream())

    def read(self, ty, starts, lens, n=None, fill=7.0):
        torch = torch_cuda()
        n = starts[-1] if n is None else n
        k = torch.full((max(n, 1), self.kv, self.dim), fill, dtype=_t(ty), device="cuda")
        v = torch.full_like(k, fill)
        s, l = _i32(starts), _i32(lens)
        self.dev.kv4_read(self.c, ty, n, len(lens), s.data_ptr(), l.data_ptr(), k.data_ptr(), self.kv * self.dim,
                          v.data_ptr(), self.kv * self.dim, stream())
        sync()
        return _host(k)[:n], _host(v)[:n]

    def all(self, lens):
        """f64 keys and values of every slot, a list of [n][kv][dim] per sequence."""
        starts = np.concatenate([[0], np.cumsum(lens)])
        k, v = self.read(aa.F32, starts, lens)
        return [(k[a:b], v[a:b]) for a, b in zip(starts[:-1], starts[1:])]


def _starts(rows):
    return np.concatenate([[0], np.cumsum(rows)]).astype(np.int64)


def _kv(gen, n, kv, dim):
    k = gen.standard_normal((n, kv, dim)) * np.exp(0.7 * gen.standard_normal((kv, dim))) + gen.standard_normal((kv, dim))
    return k.astype(np.float32), gen.standard_normal((n, kv, dim)).astype(np.float32)


def _filled(gen, dim, kv, lens, ty=aa.F32, max_pages=None, spare=3):
    c = Cache(gen, dim, kv, len(lens), max_pages or max(1, max(-(-n // 64) for n in lens)), spare)
    if sum(lens):
        k, v = _kv(gen, sum(lens), kv, dim)
        c.append(ty, _dev(k, ty), _dev(v, ty), _starts(lens), lens)
    return c


# dim, kv heads, steps of (rows of each sequence): appended one after the other
APPENDS = [
    (128, 2, [[1], [1], [62], [1], [100]]),
    (64, 3, [[5, 0, 33], [1, 1, 1], [31, 200, 0]]),
    (256, 1, [[17, 15], [64, 1]]),
    (128, 8, [[130, 1, 0, 64]]),
]


@pytest.mark.parametrize("ty", [aa.F32, aa.F16, aa.BF16], ids=NAMES.get)
@pytest.mark.parametrize("case", APPENDS, ids=lambda c: f"d{c[0]}k{c[1]}s{len(c[2])}")
def test_append_and_read(case, ty):
    dim, kv, steps = case
    gen = np.random.default_rng(dim + kv)
    n_seq = len(steps[0])
    total = [sum(s[b] for s in steps) for b in range(n_seq)]
    c = Cache(gen, dim, kv, n_seq, max(-(-t // 64) for t in total))
    lens = np.zeros(n_seq, np.int64)
    want = [([], []) for _ in range(n_seq)]
    rope = aa.Rope(dim if kv != 8 else dim // 2, base=10000.0, layout="interleaved" if kv == 3 else "half")
    f, mag = rope.table()
    for i, rows in enumerate(steps):
        st, lens = _starts(rows), lens + rows
        k, v = _kv(gen, st[-1], kv, dim)
        dk, dv = _dev(k, ty), _dev(v, ty)
        hk, hv = _host(dk), _host(dv)
        if i % 2 == 0:
            pos = gen.integers(0, 200000, st[-1])
            hk = plain.rotate(hk, pos, f, mag, kv == 3)
            c.append(ty, dk, dv, st, lens, rope, pos)
        else:
            c.append(ty, dk, dv, st, lens)
        ks, vs = plain.pair_stands_for(hk.astype(np.float32), hv.astype(np.float32))
        for b in range(n_seq):
            want[b][0].append(ks[st[b]:st[b + 1]])
            want[b][1].append(vs[st[b]:st[b + 1]])
    for out in (aa.F32, ty):
        got = c.read(out, _starts(total), total)
        for which in (0, 1):
            w = np.concatenate([x for b in range(n_seq) for x in want[b][which]])
            exact = _host(_dev(w.astype(np.float32), out))
            assert np.array_equal(got[which], exact), np.abs(got[which] - exact).max()


def test_page_layout():
    """The documented addresses of codes and scales, byte by byte."""
    gen = np.random.default_rng(9)
    bits = (6, 22, 2, 18, 14, 30, 10, 26)
    for dim in (64, 128, 256):
        groups, quad = dim // 32, min(dim // 32, 4)
        c = Cache(gen, dim, 2, 1, 1, spare=0)
        k, v = _kv(gen, 64, 2, dim)
        c.append(aa.F32, _dev(k), _dev(v), [0, 64], [64])
        sync()
        page = c.pages.cpu().numpy().reshape(2, 80 * dim)
        words, halfs = page.view(np.uint32), page.view(np.float16).astype(np.float64)
        (kd, km, kq), (vd, vm, vq) = plain.quantise(k), plain.quantise(v)
        kq, vq = kq.reshape(64, 2, dim).astype(np.int64), vq.reshape(64, 2, dim).astype(np.int64)

        def code(w, j):
            w = int(w)
            return ((w >> bits[j]) | (w << (32 - bits[j]))) & 15
        for h in range(2):
            for t in (0, 1, 15, 16, 37, 63):
                for d in (0, 7, 8, 31, 32, dim - 1):
                    g = d // 32
                    kw = t // 16 * 2 * dim + g // quad * 64 * quad + (16 * (d % 32 // 8) + t % 16) * quad + g % quad
                    assert code(words[h, kw], d % 8) == kq[t, h, d]
                    rg, hi, lo = t % 16 // 4, t % 32 // 16, t % 4
                    vw = 8 * dim + t // 32 * 4 * dim + d // 64 * 256 + (16 * rg + d % 16) * 4 + d // 16 % 4
                    assert code(words[h, vw], 4 * hi + lo) == vq[t, h, d]
                    ks = 32 * dim + t * 2 * groups + g
                    assert halfs[h, ks] == kd[t, h, g] and halfs[h, ks + groups] == km[t, h, g]
                    vs = 36 * dim + t // 32 * 64 * groups + g * 32 + rg * 8 + hi * 4 + lo
                    assert halfs[h, vs] == vd[t, h, g] and halfs[h, vs + 32 * groups] == vm[t, h, g]


def test_append_of_ties_constants_and_values_beyond_the_format():
    gen = np.random.default_rng(3)
    x = np.zeros((9, 1, 64), np.float32)
    x[0, 0, :32] = np.arange(32) / 2.0 % 15.5            # exact halves: ties to even
    x[0, 0, 32:] = 3.25                                   # a constant group
    x[1, 0] = gen.standard_normal(64) * 1e-7              # steps at the finest quantum
    x[2, 0] = gen.standard_normal(64) * 500
    x[3, 0, 3] = np.nan
    x[4, 0, 40] = np.inf
    x[5, 0, 3] = -70000.0                                 # a minimum beyond f16
    x[6, 0, 3] = 4000.0                                   # a step above 254
    x[7, 0] = -0.0
    x[8, 0] = np.float32(1 + 2.0 ** -11) * (1 + np.arange(64) % 2)   # the f16 minimum lies above or below
    other = gen.standard_normal((9, 1, 64)).astype(np.float32)
    for k, v in ((x, x), (x, other), (other, x)):
        c = Cache(gen, 64, 1, 1, 1)
        c.append(aa.F32, _dev(k), _dev(v), [0, 9], [9])
        got = c.read(aa.F32, [0, 9], [9])
        for g, want in zip(got, plain.pair_stands_for(k, v)):
            assert np.isnan(want[3:7]).all() and np.isfinite(want[:3]).all() and np.isfinite(want[7:]).all()
            assert np.array_equal(g, want.astype(np.float32).astype(np.float64), equal_nan=True)


def test_append_ties_that_lost_bits_break():
    """Values whose difference from the minimum is a tie after its rounding to
    f32 but not before: the lost bits decide, not evenness."""
    gen = np.random.default_rng(2)
    dim = 64
    tiny = np.float32(2.0 ** -24)
    rows = []
    # Minimum 2^-24, d = 1: n + 1/2 less 2^-24 goes down.  Minimum -2^-24,
    # d = 1 + 2^-6 (the 7-bit step above 1): (n + 1/2) d and 2^-24 goes up.
    # Both differences round to the tie from 2 on (ulp 2^-22).
    for m, d in ((tiny, 1.0), (-tiny, 1.015625)):
        g = np.full(32, m, np.float32)
        g[1] = 15.0
        for n in range(2, 14):
            g[n] = (n + 0.5) * d
        rows.append(np.concatenate([g, gen.permutation(g)]))
    x = np.stack(rows)[:, None]
    d, _, q = plain.quantise(x)
    assert (d[0] == 1.0).all() and (d[1] == 1.015625).all()
    assert (q[0, 0, 0, 2:14] == np.arange(2, 14)).all() and (q[1, 0, 0, 2:14] == np.arange(3, 15)).all()
    c = Cache(gen, dim, 1, 1, 1)
    c.append(aa.F32, _dev(x), _dev(x), [0, 2], [2])
    k, v = c.all([2])[0]
    want = plain.stands_for(x).astype(np.float32)  # d q + m rounded once, as it is read (3 + 2^-24 is no f32)
    assert (k == want).all() and (v == want).all()


def test_append_leaves_the_rest_alone():
    """Slots before and behind the new rows, other pages, and slots that the
    table does not have (page -1, a page past the pool, more slots than pages)."""
    gen = np.random.default_rng(21)
    c = _filled(gen, 128, 2, [100, 70], max_pages=3)
    before = c.all([100, 70])
    c2 = c.pages.clone()
    table = c.host_table.copy()
    table[0, 1], table[1, 1] = -1, c.pool
    c.set_table(table)
    k, v = _kv(gen, 100, 2, 128)
    c.append(aa.F32, _dev(k), _dev(v), [0, 50, 100], [150, 250])  # slots 100..149 and 200..249
    sync()
    c.set_table(c.host_table)
    after = c.all([100, 70])
    for (a, b), (d, e) in zip(before, after):
        assert np.array_equal(a, d) and np.array_equal(b, e)
    changed = (c2 != c.pages).any(1).cpu().numpy().nonzero()[0]
    assert set(changed) <= {int(c.host_table[0, 2])}  # slots 128..149 alone are in a page of the pool
    got = c.read(aa.F32, [0, 2], [3 * 64 + 2, 0][:1], n=2)
    assert np.isnan(got[0]).all()  # past max_pages
    k0, v0 = _kv(gen, 5, 2, 128)
    c.append(aa.F32, _dev(k0), _dev(v0), [0, 5, 5], [2, 0])   # three rows lie below slot 0
    g, _ = c.read(aa.F32, [0, 2, 2], [2, 0])
    assert np.array_equal(g, plain.stands_for(k0)[3:].astype(np.float32).astype(np.float64))


# ---- attention ---------------------------------------------------------------

def _bounds(ty, n, pv, sk, out, lse):
    s = 2.0 ** -19 * sk
    sums = (n / 16 + 64) * U
    w = 2 * s + 2.0 ** -20 + sums + (0 if ty == aa.F32 else 2 * 2.0 ** -11)
    b_out = w[..., None] * pv + HALF[ty] * np.abs(out) + TINY[ty]
    with np.errstate(invalid="ignore"):
        b_lse = s + 2.0 ** -20 + sums + U * np.abs(lse)
    return b_out, b_lse


def _attend(c, ty, q, starts, lens, heads, scale, window=0, max_rows=None, want_lse=True, out_stride=None, many=False):
    """many: in a batch of at least 80 columns a sequence and 20480 in all, most
    of them rows behind the last sequence, as the kernel for many rows takes."""
    torch = torch_cuda()
    if many:
        n = q.shape[0]
        q = torch.cat([q, q.new_zeros((max(80, -(-20480 // heads)), q.shape[1]))])
        out, lse = _attend(c, ty, q, starts, lens, heads, scale, window, max(80, max_rows or int(np.diff(starts).max())),
                           want_lse, out_stride)
        assert (out[n:] == 7).all() and (lse[n:] == 7).all()
        return out[:n], lse[:n]
    n, dim = q.shape[0], c.dim
    rows = np.diff(starts)
    st, ln = _i32(starts), _i32(lens)
    stride = out_stride or heads * dim
    out = torch.full((n, stride), 7.0, dtype=_t(ty), device="cuda")
    lse = torch.full((n, heads), 7.0, device="cuda")
    mr = max_rows or max(1, int(rows.max()))
    work = torch.full((c.dev.kv4_attention_work_bytes(c.c, heads, n, len(lens), mr),), 0xFF, dtype=torch.uint8, device="cuda")
    c.dev.kv4_attention(c.c, ty, q.data_ptr(), q.stride(0), heads, n, len(lens), st.data_ptr(), mr, ln.data_ptr(), scale,
                        out.data_ptr(), stride, work.data_ptr(), stream(), window=window,
                        lse=lse.data_ptr() if want_lse else 0)
    sync()
    return out, lse


def _check(c, ty, q, starts, lens, heads, scale, window, out, lse, kvs=None):
    kvs = kvs or c.all(lens)
    hq = _host(q)[:, :heads * c.dim].reshape(-1, heads, c.dim)
    ho, hl = _host(out)[:, :heads * c.dim].reshape(-1, heads, c.dim), _host(lse)
    for b, n in enumerate(lens):
        r0, r1 = starts[b], starts[b + 1]
        rows = min(r1 - r0, n)
        for r in range(r0, r1 - rows):  # rows below slot 0 see nothing
            assert np.all(ho[r] == 0) and np.all(hl[r] == -np.inf)
        if not rows:
            continue
        k, v = kvs[b]
        want, wl, pv, sk = plain.attend(hq[r1 - rows:r1], k, v, scale, window)
        bo, bl = _bounds(ty, n, pv, sk, want, wl)
        eo = np.abs(ho[r1 - rows:r1] - want)
        assert np.all(eo <= bo), (b, np.max(eo / bo))
        with np.errstate(invalid="ignore"):
            el = np.where(wl == hl[r1 - rows:r1], 0, np.abs(hl[r1 - rows:r1] - wl))
            assert np.all(el <= np.where(np.isfinite(bl), bl, 0)), (b, np.nanmax(el / bl))


ATTENTION = [
    # dim, heads, kv, rows, lens, window
    (128, 4, 1, [1], [1], 0),
    (128, 32, 8, [1, 1, 1, 1], [17, 0, 64, 65], 0),
    (128, 32, 8, [1], [1000], 0),
    (128, 8, 8, [1, 1], [31, 300], 0),                 # a query head per kv head
    (128, 5, 1, [1, 1], [129, 33], 0),                 # an odd group
    (128, 16, 1, [1], [2500], 0),
    (128, 40, 1, [1, 1], [100, 700], 0),               # more heads than a tile
    (64, 6, 3, [1, 1], [63, 500], 0),
    (64, 24, 1, [2, 1], [5, 200], 0),
    (256, 8, 4, [1, 1], [16, 400], 0),
    (256, 2, 1, [3], [3], 0),
    (128, 8, 2, [1, 1, 1], [15, 400, 64], 1),          # only itself
    (128, 8, 2, [1, 1], [700, 90], 64),
    (128, 8, 2, [2, 7, 3], [130, 7, 66], 0),           # several rows each
    (128, 8, 2, [5, 0, 4], [3, 10, 0], 0),             # rows below slot 0, none, an empty sequence
    (128, 8, 2, [16], [16], 0),
    (128, 8, 2, [33, 64, 1], [33, 200, 300], 0),
    (128, 4, 1, [130], [130], 0),
    (128, 8, 2, [130, 20], [257, 20], 33),
    (128, 3, 3, [70], [70], 0),
    (128, 12, 1, [50], [77], 0),
    (64, 4, 2, [150, 31], [150, 160], 0),
    (64, 2, 2, [129], [200], 17),
    (256, 4, 2, [70, 1], [70, 129], 0),
    (256, 2, 2, [130], [190], 0),
]


@pytest.mark.parametrize("ty", [aa.F32, aa.BF16, aa.F16], ids=NAMES.get)
@pytest.mark.parametrize("case", ATTENTION, ids=lambda c: f"d{c[0]}h{c[1]}k{c[2]}r{'_'.join(map(str, c[3]))}n{'_'.join(map(str, c[4]))}w{c[5]}")
@pytest.mark.parametrize("many", [False, True], ids=["few", "many"])
def test_attention(case, ty, many):
    dim, heads, kv, rows, lens, window = case
    gen = np.random.default_rng(dim + heads + sum(lens))
    c = _filled(gen, dim, kv, lens, max_pages=-(-max(lens) // 64) + 1)
    st = _starts(rows)
    q = _dev(2 * gen.standard_normal((st[-1], heads * dim)).astype(np.float32), ty)
    out, lse = _attend(c, ty, q, st, lens, heads, dim ** -0.5, window, many=many)
    _check(c, ty, q, st, lens, heads, dim ** -0.5, window, out, lse)
    again, lse2 = _attend(c, ty, q, st, lens, heads, dim ** -0.5, window, max_rows=max(1, max(rows)), many=many)
    assert (again == out).all() and (lse2 == lse).all()


# dim, heads, kv, rows, lens, window: shares of a long axis, a sequence in
# parts of several workgroups and several sequences in one, over 64 of them.
SHARES = [
    (64, 4, 1, [1], [9001], 0),
    (64, 4, 2, [3, 1], [4100, 33], 2000),
    (256, 2, 1, [1, 1], [5000, 1], 0),
    (128, 4, 4, [5], [3300], 0),
    (64, 2, 1, [1, 2, 0] * 30, [(37 * i) % 300 for i in range(90)], 0),
    (128, 8, 1, [1] * 129, [2000 if i == 70 else i % 7 for i in range(129)], 50),
]


@pytest.mark.parametrize("ty", [aa.F32, aa.BF16], ids=NAMES.get)
@pytest.mark.parametrize("case", SHARES, ids=lambda c: f"d{c[0]}h{c[1]}k{c[2]}s{len(c[3])}n{max(c[4])}w{c[5]}")
def test_attention_shares_and_parts(case, ty):
    dim, heads, kv, rows, lens, window = case
    gen = np.random.default_rng(dim + len(rows))
    c = _filled(gen, dim, kv, lens, max_pages=-(-max(lens) // 64))
    st = _starts(rows)
    q = _dev(2 * gen.standard_normal((st[-1], heads * dim)).astype(np.float32), ty)
    out, lse = _attend(c, ty, q, st, lens, heads, dim ** -0.5, window)
    _check(c, ty, q, st, lens, heads, dim ** -0.5, window, out, lse)
    # A bound, no size; the axis is cut by it.
    out, lse = _attend(c, ty, q, st, lens, heads, dim ** -0.5, window, max_rows=2 ** 31 - 1)
    _check(c, ty, q, st, lens, heads, dim ** -0.5, window, out, lse)


@pytest.mark.parametrize("rows,lens,many", [([1, 1], [200, 40], False), ([40, 3], [100, 40], False),
                                            ([100, 3], [130, 40], True)], ids=["decode", "prompt", "many"])
def test_attention_strides_types_of_rows_and_untouched_memory(rows, lens, many):
    """Rows at odd strides, rows behind the last sequence, max_rows that is not
    the longest, and no lse wanted."""
    torch = torch_cuda()
    gen = np.random.default_rng(8)
    heads, kv, dim = 6, 2, 128
    for ty in (aa.F32, aa.BF16):
        c = _filled(gen, dim, kv, lens)
        st = _starts(rows)
        wide = heads * dim + 3
        q = _dev(gen.standard_normal((st[-1] + 2, wide)).astype(np.float32), ty)
        out, lse = _attend(c, ty, q, st, lens, heads, 0.2, out_stride=wide, many=many)
        n = int(st[-1])
        assert (out[n:] == 7).all() and (out[:, heads * dim:] == 7).all() and (lse[n:] == 7).all()
        _check(c, ty, q, st, lens, heads, 0.2, 0, out, lse)
        for mr in (1, 17, 1000):
            o2, l2 = _attend(c, ty, q, st, lens, heads, 0.2, max_rows=mr, out_stride=wide, many=many)
            for b, r in enumerate(rows):  # rows past max_rows: NaN
                over = slice(int(st[b]) + min(r, max(mr, 80) if many else mr), int(st[b + 1]))
                assert torch.isnan(o2[over, :heads * dim]).all() and torch.isnan(l2[over]).all()
                o2[over], l2[over] = out[over], lse[over]
            _check(c, ty, q, st, lens, heads, 0.2, 0, o2, l2)
        o3, l3 = _attend(c, ty, q, st, lens, heads, 0.2, out_stride=wide, want_lse=False, many=many)
        assert (o3 == out).all() and (l3 == 7).all()


@pytest.mark.parametrize("rows,many", [(1, False), (40, False), (40, True)], ids=["decode", "prompt", "many"])
@pytest.mark.parametrize("ty", [aa.F32, aa.F16], ids=NAMES.get)
def test_attention_scales_of_the_values(rows, many, ty):
    """One-hot and flat softmaxes, tiny and large keys and values, zero queries,
    constant keys, a slot whose weight dwarfs the others' with values near 0."""
    gen = np.random.default_rng(31)
    dim, heads, kv, n = 128, 4, 1, 150
    for kk, vv, qq, scale in ((1.0, 1.0, 8.0, 1.0), (1e-4, 1e-5, 1.0, 1.0), (60.0, 200.0, 0.05, 0.1), (1.0, 1.0, 0.0, 1.0),
                              (0.0, 1.0, 1.0, 1.0), (1.0, 1e-3, 1e-4, 1.0), (1.0, 1.0, 100.0, 1e-3), (1.0, 1.0, 1.0, -0.1)):
        c = Cache(gen, dim, kv, 1, 3)
        k, v = _kv(gen, n, kv, dim)
        k, v = k * np.float32(kk), v * np.float32(vv)
        k[0] *= 3
        v[0] *= np.float32(1e-3)
        c.append(aa.F32, _dev(k), _dev(v), [0, n], [n])
        q = _dev((qq * gen.standard_normal((rows, heads * dim))).astype(np.float32), ty)
        out, lse = _attend(c, ty, q, [0, rows], [n], heads, scale, many=many)
        _check(c, ty, q, [0, rows], [n], heads, scale, 0, out, lse)


@pytest.mark.parametrize("rows,many", [(1, False), (40, False), (40, True)], ids=["decode", "prompt", "many"])
@pytest.mark.parametrize("ty", [aa.F32, aa.BF16], ids=NAMES.get)
def test_masked_slots_never_matter_and_seen_ones_always(rows, many, ty):
    """Slots behind the length and before the window hold NaN scales; a NaN or
    infinity in a query, a NaN key in sight and a page that is not there make
    the rows that see them NaN, and no others."""
    gen = np.random.default_rng(41)
    dim, heads, kv = 128, 8, 2
    lens = [90 + rows, 20 + rows]
    c = _filled(gen, dim, kv, lens, max_pages=4)
    kvs = c.all(lens)
    bad_k = np.full((30, kv, dim), np.nan, np.float32)
    c.append(aa.F32, _dev(bad_k), _dev(bad_k), [0, 30, 30], [30, 0])  # slots 0..29 of sequence 0
    st = np.array([0, rows, 2 * rows])
    host = gen.standard_normal((2 * rows, heads * dim)).astype(np.float32)
    q = _dev(host, ty)
    # Every row of sequence 0 sees slots 61 and up at least, none below 30.
    out, lse = _attend(c, ty, q, st, lens, heads, 0.1, window=60, many=many)
    _check(c, ty, q, st, lens, heads, 0.1, 60, out, lse, kvs)
    out, lse = _attend(c, ty, q, st, lens, heads, 0.1, many=many)
    assert np.isnan(_host(out)[:rows]).all() and np.isnan(_host(lse)[:rows]).all()
    assert np.isfinite(_host(out)[rows:]).all()
    host2 = host.copy()
    host2[0, 3] = np.nan
    host2[rows, dim + 5] = np.inf
    q2 = _dev(host2, ty)
    out, lse = _attend(c, ty, q2, st, lens, heads, 0.1, window=60, many=many)
    o = _host(out).reshape(2 * rows, heads, dim)
    assert np.isnan(o[0, 0]).all() and np.isnan(o[rows, 1]).all()
    o[0, 0], o[rows, 1] = 0, 0
    assert np.isfinite(o).all()
    for page in (-1, c.pool, 1 << 30):
        table = c.host_table.copy()
        table[1, 0] = page
        c.set_table(table)
        out, lse = _attend(c, ty, q, st, lens, heads, 0.1, window=60, many=many)
        assert np.isnan(_host(out)[rows:]).all() and np.isfinite(_host(out)[:rows]).all()
    c.set_table(c.host_table)
    long = [4 * 64 + rows + 70, lens[1]]  # longer than the table: its rows see slots past it
    out, _ = _attend(c, ty, q, st, long, heads, 0.1, window=60, many=many)
    assert np.isnan(_host(out)[:rows]).all() and np.isfinite(_host(out)[rows:]).all()


def test_attention_bad_row_starts_are_bounded():
    """Row starts that fall, point past n_rows or below 0 read as empty or cut;
    no row outside [0, n_rows) is touched."""
    gen = np.random.default_rng(6)
    c = _filled(gen, 64, 1, [50, 50, 50])
    q = _dev(gen.standard_normal((4, 128)).astype(np.float32))
    out, lse = _attend(c, aa.F32, q, [-3, 2, 1, 900], [50, 50, 50], 2, 0.1, max_rows=4)
    # Row 1 is also sequence 2's (it starts there); row 0 is sequence 0's alone, one before its last.
    ok, ol = out.clone(), lse.clone()
    k, v = c.all([50, 50, 50])[0]
    want, wl, pv, sk = plain.attend(_host(q)[:2].reshape(2, 2, 64), k, v, 0.1)
    bo, bl = _bounds(aa.F32, 50, pv, sk, want, wl)
    assert np.all(np.abs(_host(ok)[0].reshape(2, 64) - want[0]) <= bo[0]) and np.all(np.abs(_host(ol)[0] - wl[0]) <= bl[0])
    assert np.isfinite(_host(out)).all() and (lse != 7).all()


def test_cache_beyond_32_bit_offsets():
    """Pages whose bytes lie past 2^32 in the pool."""
    torch = torch_cuda()
    gen = np.random.default_rng(2)
    dim, kv, lens = 128, 8, [150, 70]
    c = Cache(gen, dim, kv, 2, 3, spare=(5 << 30) // (80 * dim * kv), fill=0)
    table = c.pool - 1 - np.arange(6, dtype=np.int32).reshape(2, 3) * 7
    c.set_table(table)
    k, v = _kv(gen, 220, kv, dim)
    c.append(aa.F32, _dev(k), _dev(v), _starts(lens), lens)
    got = c.all(lens)
    assert np.array_equal(np.concatenate([g[0] for g in got]), plain.stands_for(k).astype(np.float32))
    for rows in ([1, 1], [70, 40]):
        st = _starts(rows)
        q = _dev(gen.standard_normal((st[-1], 16 * dim)).astype(np.float32))
        out, lse = _attend(c, aa.F32, q, st, lens, 16, 0.1)
        _check(c, aa.F32, q, st, lens, 16, 0.1, 0, out, lse, got)
    del c
    torch.cuda.empty_cache()


# ---- slot weights and eviction -----------------------------------------------

@pytest.mark.parametrize("ty", [aa.F32, aa.BF16], ids=NAMES.get)
@pytest.mark.parametrize("case", ATTENTION[:12] + ATTENTION[13:15] + ATTENTION[16:19] + ATTENTION[20:24],
                         ids=lambda c: f"d{c[0]}h{c[1]}k{c[2]}r{'_'.join(map(str, c[3]))}n{'_'.join(map(str, c[4]))}w{c[5]}")
def test_slot_weights(case, ty):
    dim, heads, kv, rows, lens, window = case
    torch = torch_cuda()
    gen = np.random.default_rng(dim + heads + sum(lens))
    c = _filled(gen, dim, kv, lens)
    st, scale = _starts(rows), dim ** -0.5
    q = _dev(2 * gen.standard_normal((st[-1], heads * dim)).astype(np.float32), ty)
    _, lse = _attend(c, ty, q, st, lens, heads, scale, window)
    stride = max(lens) - 3 if max(lens) > 100 else max(lens) + 5
    first = gen.random((len(lens), kv, stride)).astype(np.float32)
    s, l = _i32(st), _i32(lens)
    hq, hl = _host(q).reshape(-1, heads, dim), _host(lse)
    results = []
    for acc_in in ("other", "same", "none"):
        a = _dev(first)
        out = a if acc_in == "same" else torch.full_like(a, 7.0)
        c.dev.kv4_weigh(c.c, ty, q.data_ptr(), heads * dim, heads, int(st[-1]), len(lens), s.data_ptr(),
                        max(1, max(rows)), l.data_ptr(), scale, lse.data_ptr(), 0 if acc_in == "none" else a.data_ptr(),
                        out.data_ptr(), stride, stream(), window=window)
        sync()
        results.append(_host(out))
    for b, n in enumerate(lens):
        r1 = st[b + 1]
        r = min(r1 - st[b], n)
        m = min(n, stride)
        k, v = c.all(lens)[b]
        w = plain.weights(hq[r1 - r:r1], k, hl[r1 - r:r1], scale, window)[:, :m] if r else np.zeros((kv, m))
        size = np.abs(hq[r1 - r:r1]).max(initial=0) * plain.parts(k).max(initial=0) * dim * scale if n else 0.0  # at least sum |q| parts
        for got, base in zip(results, (first[b], first[b], np.zeros_like(first[b]))):
            want = base[:, :m] + w
            bound = w * (2.0 ** -19 * size + 2.0 ** -20 + (heads // kv * max(r, 1) + 8) * U) + U * np.abs(want) + 1e-30
            assert np.all(np.abs(got[b][:, :m] - want) <= bound), np.max(np.abs(got[b][:, :m] - want) / bound)
        for got, base in zip(results, (first[b], first[b], np.zeros_like(first[b]))):
            assert np.array_equal(got[b][:, m:], base[:, m:])  # slots behind the length


def test_slot_weights_with_too_small_max_rows():
    """A sequence with more rows than max_rows gives NaN, the others are right."""
    torch = torch_cuda()
    gen = np.random.default_rng(3)
    c = _filled(gen, 128, 1, [100, 80])
    q = _dev(gen.standard_normal((6, 2 * 128)).astype(np.float32))
    for rows, mr in (([5, 1], 1), ([1, 5], 4)):
        st = _starts(rows)
        _, lse = _attend(c, aa.F32, q, st, [100, 80], 2, 0.1)
        out = torch.zeros(2, 1, 128, device="cuda")
        s, l = _i32(st), _i32([100, 80])
        c.dev.kv4_weigh(c.c, aa.F32, q.data_ptr(), 256, 2, 6, 2, s.data_ptr(), mr, l.data_ptr(), 0.1, lse.data_ptr(), 0,
                        out.data_ptr(), 128, stream())
        sync()
        bad = 0 if rows[0] == 5 else 1
        o = _host(out)[:, 0]
        assert np.isnan(o[bad, :[96, 76][bad]]).all() and np.abs(o[1 - bad].sum() - 2) < 1e-4


EVICTS = [
    # dim, kv, lens, keep, first, recent
    (128, 2, [200, 64, 10, 0], 64, 4, 16),
    (64, 3, [1000, 333], 100, 0, 0),
    (256, 1, [300], 65, 1, 64),         # nothing in between
    (128, 1, [5000], 1500, 4, 100),
    (64, 1, [130, 131, 129], 129, 0, 129),
    (64, 2, [70, 1], 1, 0, 0),
]


@pytest.mark.parametrize("case", EVICTS, ids=lambda c: f"d{c[0]}k{c[1]}n{'_'.join(map(str, c[2]))}to{c[3]}")
@pytest.mark.parametrize("weights", ["spread", "ties", "odd"])
def test_evict(case, weights):
    dim, kv, lens, keep, first, recent = case
    torch = torch_cuda()
    gen = np.random.default_rng(keep + dim)
    c = _filled(gen, dim, kv, lens)
    kvs = c.all(lens)
    n_seq, stride = len(lens), max(lens) + (7 if weights != "odd" else -9 if max(lens) > 100 else 0)
    acc = np.exp(2 * gen.standard_normal((n_seq, kv, stride))).astype(np.float32)
    if weights == "ties":
        acc = np.round(acc).astype(np.float32)
    if weights == "odd":  # NaN, infinities, negatives, zeros of both signs, denormals
        some = np.array([np.nan, np.inf, -np.inf, -1.0, 0.0, -0.0, 1e-40, 1e-42, 3e38, 1.0], np.float32)
        acc = some[gen.integers(0, len(some), acc.shape)]
    dst = Cache(gen, dim, kv, n_seq, -(-keep // 64) + 1, spare=0)
    new_len = _i32([99] * n_seq)
    idx = _i32(np.full((n_seq, kv, keep), 99))
    out = torch.full((n_seq, kv, keep), 7.0, device="cuda")
    ln, ac = _i32(lens), _dev(acc)
    c.dev.kv4_evict(c.c, n_seq, ln.data_ptr(), ac.data_ptr(), stride, keep, first, recent, dst.c, new_len.data_ptr(),
                    idx.data_ptr(), out.data_ptr(), stream())
    sync()
    kept = [min(n, keep) for n in lens]
    assert new_len.cpu().tolist() == kept
    hi, ho = idx.cpu().numpy(), out.cpu().numpy()
    new = dst.all(kept)
    for b, n in enumerate(lens):
        for h in range(kv):
            want = plain.keep_slots(acc[b, h], n, keep, first, recent)
            assert np.array_equal(hi[b, h, :kept[b]], want)
            w = np.zeros(max(n, stride), np.float32)
            w[:stride] = acc[b, h]
            assert np.array_equal(ho[b, h, :kept[b]], w[want], equal_nan=True)
            assert np.all(hi[b, h, kept[b]:] == -1) and np.all(ho[b, h, kept[b]:] == 0)
            for which in (0, 1):
                assert np.array_equal(new[b][which][:, h], kvs[b][which][want, h])


def test_evict_from_pages_that_are_not_there():
    torch = torch_cuda()
    gen = np.random.default_rng(1)
    c = _filled(gen, 64, 1, [200])
    t = c.host_table.copy()
    t[0, 0] = -1
    c.set_table(t)
    dst = Cache(gen, 64, 1, 1, 2)
    acc = _dev(np.ones((1, 1, 200), np.float32))
    idx, out, nl, ln = _i32(np.zeros(100)), torch.zeros(100, device="cuda"), _i32([0]), _i32([200])
    c.dev.kv4_evict(c.c, 1, ln.data_ptr(), acc.data_ptr(), 200, 100, 0, 40, dst.c, nl.data_ptr(), idx.data_ptr(),
                    out.data_ptr(), stream())
    k, v = dst.read(aa.F32, [0, 100], [100])
    assert np.isnan(k[:60]).all() and np.isnan(v[:60]).all() and np.isfinite(k[60:]).all()


# ---- together ------------------------------------------------------------------

def _layer(gen, heads, kv, dim, hidden):
    from aspida_amd import synth
    torch = torch_cuda()
    dev = aa.DeviceOps()
    mats = {}
    for name, kind, o, i in (("qk", aa.Q4_K, (heads + kv) * dim, hidden), ("v", aa.Q6_K, kv * dim, hidden),
                             ("o", aa.Q4_K, hidden, heads * dim)):
        w = synth.weight_np(kind, o, i, gen)
        p = torch.empty(dev.packed_bytes(kind, i, o), dtype=torch.uint8, device="cuda")
        dw = _dev(w)
        dev.pack(kind, dw.data_ptr(), i, o, p.data_ptr(), stream())
        sync()
        mats[name] = (kind, p, i, o)
    return mats


class Step:
    """A decoder layer's attention for B lanes on this library alone: q|k and v
    products, rope on q, append (keys rotated), attention, o product."""

    def __init__(self, gen, lanes, heads=8, kv=2, dim=128, hidden=1024, max_pages=4):
        torch = torch_cuda()
        self.mats = _layer(gen, heads, kv, dim, hidden)
        self.c = Cache(gen, dim, kv, lanes, max_pages)
        self.rope = aa.Rope(dim, base=500000.0)
        self.sizes = lanes, heads, kv, dim, hidden
        e = lambda *s: torch.empty(*s, device="cuda")  # noqa: E731
        self.x = _dev(gen.standard_normal((lanes, hidden)).astype(np.float32))
        self.qk, self.v, self.att, self.y = e(lanes, (heads + kv) * dim), e(lanes, kv * dim), e(lanes, heads * dim), e(lanes, hidden)
        self.len, self.pos = _i32([0] * lanes), _i32([0] * lanes)
        self.lse = e(lanes, heads)
        self.work = torch.empty(self.c.dev.kv4_attention_work_bytes(self.c.c, heads, lanes, lanes, 1), dtype=torch.uint8,
                                device="cuda")

    def run(self):
        lanes, heads, kv, dim, hidden = self.sizes
        dev, sp, row = self.c.dev, stream(), (heads + kv) * dim
        for name, x, y in (("qk", self.x, self.qk), ("v", self.x, self.v)):
            kind, p, i, o = self.mats[name]
            dev.matmul_packed(kind, p.data_ptr(), i, o, lanes, x.data_ptr(), y.data_ptr(), sp)
        q, k = self.qk.data_ptr(), self.qk.data_ptr() + 4 * heads * dim
        dev.kv4_append(self.c.c, aa.F32, k, row, self.v.data_ptr(), kv * dim, lanes, lanes, 0, self.len.data_ptr(),
                       self.rope, self.pos.data_ptr(), sp)
        dev.rope(self.rope, aa.F32, q, row, lanes, heads, dim, self.pos.data_ptr(), q, row, sp)
        dev.kv4_attention(self.c.c, aa.F32, q, row, heads, lanes, lanes, 0, 1, self.len.data_ptr(), dim ** -0.5,
                          self.att.data_ptr(), heads * dim, self.work.data_ptr(), sp, lse=self.lse.data_ptr())
        kind, p, i, o = self.mats["o"]
        dev.matmul_packed(kind, p.data_ptr(), i, o, lanes, self.att.data_ptr(), self.y.data_ptr(), sp)


def _steps(step, run, n):
    """n tokens; the outputs of each."""
    got = []
    for t in range(n):
        step.len.fill_(t + 1)
        step.len[0] = t + 1 + 60  # lane 0 starts at slot 60
        step.pos.copy_(step.len - 1)
        step.x.copy_(step.inputs[t])
        run()
        sync()
        got.append((step.y.clone(), step.att.clone()))
    return got


def test_decode_steps_eager_and_captured():
    """Tokens of a layer one after the other, against the plain form over what
    the cache holds; then the same tokens by replays of a graph captured from
    one step, with eager work between them: the same bits."""
    torch = torch_cuda()
    gen = np.random.default_rng(77)
    step = Step(gen, 3)
    lanes, heads, kv, dim, hidden = step.sizes
    n = 9
    step.inputs = [_dev(gen.standard_normal((lanes, hidden)).astype(np.float32)) for _ in range(n)]
    kf, vf = _kv(gen, 60, kv, dim)
    step.c.append(aa.F32, _dev(kf), _dev(vf), [0, 60, 60, 60], [60, 0, 0])
    eager = _steps(step, step.run, n)
    lens = [n + 60, n, n]
    kvs = step.c.all(lens)
    q = _host(step.qk)[:, :heads * dim].reshape(lanes, heads, dim)
    for b in range(lanes):
        want, wl, pv, sk = plain.attend(q[b:b + 1], *kvs[b], dim ** -0.5)
        bo, _ = _bounds(aa.F32, lens[b], pv, sk, want, wl)
        assert np.all(np.abs(_host(eager[-1][1])[b].reshape(heads, dim) - want[0]) <= bo[0])
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step.run()
    sync()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step.run()

    def replay():
        graph.replay()
        torch.ones(1000, device="cuda").sum()
    again = _steps(step, replay, n)
    for (a, b), (c, d) in zip(eager, again):
        assert torch.equal(a, c) and torch.equal(b, d)


def test_prompt_then_tokens_then_eviction():
    """A prompt in two chunks gives the rows one call gives; weights are taken
    from the last rows, the cache is shrunk, and attention over the kept slots
    matches the plain form over them."""
    torch = torch_cuda()
    gen = np.random.default_rng(12)
    dim, heads, kv, n = 128, 8, 2, 300
    k, v = _kv(gen, n, kv, dim)
    q = _dev(gen.standard_normal((n, heads * dim)).astype(np.float32))
    whole = Cache(gen, dim, kv, 1, 5)
    whole.append(aa.F32, _dev(k), _dev(v), [0, n], [n])
    out, lse = _attend(whole, aa.F32, q, [0, n], [n], heads, 0.1)
    parts = Cache(gen, dim, kv, 1, 5)
    for a, b in ((0, 170), (170, n)):
        parts.append(aa.F32, _dev(k[a:b]), _dev(v[a:b]), [0, b - a], [b])
        o, l = _attend(parts, aa.F32, q[a:b].contiguous(), [0, b - a], [b], heads, 0.1)
        _check(parts, aa.F32, q[a:b], [0, b - a], [b], heads, 0.1, 0, o, l)
        _check(whole, aa.F32, q[a:b], [0, b - a], [b], heads, 0.1, 0, out[a:b], lse[a:b])
    acc = torch.zeros(1, kv, 320, device="cuda")
    last, st, ln = q[-32:].contiguous(), _i32([0, 32]), _i32([n])
    ls = lse[-32:].contiguous()
    whole.dev.kv4_weigh(whole.c, aa.F32, last.data_ptr(), heads * dim, heads, 32, 1, st.data_ptr(), 32, ln.data_ptr(), 0.1,
                        ls.data_ptr(), acc.data_ptr(), acc.data_ptr(), 320, stream())
    sync()
    # Each row's weights sum to 1 per head: 32 rows x 4 heads per kv head.
    assert np.all(np.abs(_host(acc).sum(-1) - 32 * heads / kv) < 1e-3)
    keep = 100
    dst = Cache(gen, dim, kv, 1, 3)
    idx, w, nl = _i32(np.zeros((kv, keep))), torch.empty(1, kv, keep, device="cuda"), _i32([0])
    whole.dev.kv4_evict(whole.c, 1, ln.data_ptr(), acc.data_ptr(), 320, keep, 4, 32, dst.c, nl.data_ptr(), idx.data_ptr(),
                        w.data_ptr(), stream())
    kn, vn = _kv(gen, 1, kv, dim)
    nl += 1
    sync()
    dst.append(aa.F32, _dev(kn), _dev(vn), None, [keep + 1])
    q1 = q[:1].contiguous()
    o, l = _attend(dst, aa.F32, q1, [0, 1], [keep + 1], heads, 0.1)
    old = whole.all([n])[0]
    hi = idx.cpu().numpy().reshape(kv, keep)
    kk = np.stack([old[0][hi[h], h] for h in range(kv)], 1)
    vv = np.stack([old[1][hi[h], h] for h in range(kv)], 1)
    kvs = [(np.concatenate([kk, plain.stands_for(kn)]), np.concatenate([vv, plain.stands_for(vn)]))]
    _check(dst, aa.F32, q1, [0, 1], [keep + 1], heads, 0.1, 0, o, l, kvs)


def test_calls_on_two_streams_at_once():
    """Calls with a workspace each, on streams of their own, in flight together."""
    torch = torch_cuda()
    gen = np.random.default_rng(4)
    dim, heads, kv = 128, 8, 2
    c = _filled(gen, dim, kv, [700, 500])
    q = [_dev(gen.standard_normal((2, heads * dim)).astype(np.float32)) for _ in range(2)]
    st, ln = _i32([0, 1, 2]), _i32([700, 500])
    alone = [_attend(c, aa.F32, x, [0, 1, 2], [700, 500], heads, 0.1)[0] for x in q]
    n = c.dev.kv4_attention_work_bytes(c.c, heads, 2, 2, 1)
    works = [torch.empty(n, dtype=torch.uint8, device="cuda") for _ in q]
    outs = [torch.empty(20, 2, heads * dim, device="cuda") for _ in q]
    streams = [torch.cuda.Stream() for _ in q]
    sync()
    for i in range(20):
        for x, w, o, s in zip(q, works, outs, streams):
            c.dev.kv4_attention(c.c, aa.F32, x.data_ptr(), heads * dim, heads, 2, 2, st.data_ptr(), 1, ln.data_ptr(), 0.1,
                                o[i].data_ptr(), heads * dim, w.data_ptr(), s.cuda_stream)
    sync()
    for o, a in zip(outs, alone):
        assert (o == a).all()
