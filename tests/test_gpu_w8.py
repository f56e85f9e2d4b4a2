"""Products with 8-bit integer weights on the GPU against 64 bits.

Bounds, with u = 2^-24 and h_T half a step of the type: the codes and their
sums are exact; a product converts the sum to f32 (u) and multiplies twice
(2 u): 3 u of |y|, plus h_T of it (or half a subnormal's spacing).  Gated, a
result g h u h / (1 + h^2) with h = e^-|t|/2: g and u are off by 3 u each (6),
h by 2 u (exp2, an ulp), in the numerator twice (4) and in the denominator, with
its rounding, by at most half of 4 + 1 (2.5); the sum's reciprocal by 2 u (an
ulp); four products round (4): 18.5 u.  e^t is off by |t| times what t is: g's
3 u for silu; for gelu, formed in four operations of values with up to 3 times
g's error, 13 u at most; exp2's argument rounds once more: 14 |t| u.  In all
(19 + 14 |t|) u of |result|.
"""
import numpy as np
import pytest

import aspida_amd as aa
import more_plain as plain
import oracle
from aspida_amd import synth
from gpu_helpers import stream, sync, torch_cuda
from test_gpu_kv4 import HALF, NAMES, TINY, U, _dev, _host, _t

pytestmark = pytest.mark.gpu


class Weights:
    """Random codes (all of -128 to 127 among them) and scales, packed."""

    def __init__(self, gen, in_dim, out_dim, codes=None, scale=None, spare=0):
        torch = torch_cuda()
        self.dev = aa.DeviceOps()
        self.i, self.o = in_dim, out_dim
        self.codes = gen.integers(-128, 128, (out_dim, in_dim)).astype(np.int8) if codes is None else codes
        self.scale = (np.exp(gen.standard_normal(out_dim)) / 1000).astype(np.float32) if scale is None else scale
        self.p = torch.full((self.dev.w8_bytes(in_dim, out_dim),), 0x81, dtype=torch.uint8, device="cuda")
        held = np.full((out_dim, in_dim + spare), 77, np.int8)
        held[:, :in_dim] = self.codes
        c, s = _dev(held), _dev(self.scale)
        self.dev.w8_pack(c.data_ptr(), in_dim + spare, s.data_ptr(), in_dim, out_dim, self.p.data_ptr(), stream())
        sync()

    def work(self, n):
        torch = torch_cuda()
        return torch.full((self.dev.w8_work_bytes(n, self.i),), 0x7F, dtype=torch.uint8, device="cuda")


def _rows(gen, n, width, ty, spare):
    """Activations in rows `spare` further apart, starting at an odd element if there is room."""
    torch = torch_cuda()
    size = np.exp(0.7 * gen.standard_normal(width)) * (1 + 30 * (gen.random(width) < 0.02))
    buf = torch.full((n * (width + spare) + 1,), 3.0, dtype=_t(ty), device="cuda")
    v = buf[1 if spare else 0:][:n * (width + spare)].view(n, width + spare)[:, :width]
    v.copy_(_dev((gen.standard_normal((n, width)) * size).astype(np.float32)))
    return v


def _product(w, ty, x, spare=0, up=None, act=0, work=None):
    torch = torch_cuda()
    n = x.shape[0]
    y = torch.full((n, w.o + spare), 7.0, dtype=_t(ty), device="cuda")
    work = w.work(n) if work is None else work
    if up is None:
        w.dev.w8_matmul(w.p.data_ptr(), w.i, w.o, ty, x.data_ptr(), x.stride(0), n, y.data_ptr(), w.o + spare,
                        work.data_ptr(), stream())
    else:
        w.dev.w8_gated(w.p.data_ptr(), up.p.data_ptr(), w.i, w.o, act, ty, x.data_ptr(), x.stride(0), n, y.data_ptr(),
                       w.o + spare, work.data_ptr(), stream())
    sync()
    assert (y[:, w.o:] == 7).all()
    return y[:, :w.o]


def _check(ty, y, want):
    got = _host(y)
    bound = (3.01 * U + HALF[ty]) * np.abs(want) + TINY[ty]
    assert np.array_equal(np.isnan(got), np.isnan(want))
    with np.errstate(invalid="ignore"):
        err = np.where(np.isnan(want), 0, np.abs(got - want))
    assert np.all((err <= bound) | np.isnan(want)), np.nanmax(err / bound)


def _check_gated(ty, y, g, u, act):
    want = plain.activation(g, act) * u
    rel = (19 + 14 * np.abs(plain.gate_argument(g, act))) * U
    got = _host(y)
    bound = (rel * 1.01 + HALF[ty]) * np.abs(want) + TINY[ty]
    err = np.abs(got - want)
    assert np.all(err <= bound), np.max(err / bound)


# tokens, in, out, spare elements of a row
SIZES = [
    (1, 1, 1, 0), (1, 64, 16, 0), (1, 5, 3, 2), (2, 63, 17, 1), (3, 65, 15, 0), (1, 4096, 100, 0), (1, 20000, 33, 0),
    (4, 4096, 48, 0), (5, 4096, 48, 3), (15, 128, 64, 0), (16, 1000, 129, 0), (17, 300, 31, 5), (32, 256, 1000, 0),
    (33, 1024, 96, 0), (60, 14336, 64, 0), (64, 129, 50, 1), (65, 512, 272, 0), (100, 2048, 40, 0), (127, 192, 77, 0),
    (128, 640, 256, 0), (129, 640, 256, 0), (200, 1023, 130, 7), (300, 4096, 144, 0), (512, 64, 300, 0),
    (513, 320, 257, 0), (600, 1000, 600, 3), (1030, 384, 1, 0), (2, 300, 5000, 0), (257, 70, 2100, 0),
    (1300, 130, 1040, 0),
]


@pytest.mark.parametrize("ty", [aa.F32, aa.BF16, aa.F16], ids=NAMES.get)
@pytest.mark.parametrize("size", SIZES, ids=lambda s: f"t{s[0]}i{s[1]}o{s[2]}p{s[3]}")
def test_product(size, ty):
    n, i, o, spare = size
    gen = np.random.default_rng(n + i + o)
    w = Weights(gen, i, o, spare=spare)
    x = _rows(gen, n, i, ty, spare)
    _check(ty, _product(w, ty, x, spare), plain.product8(_host(x), w.codes, w.scale))


@pytest.mark.parametrize("ty", [aa.F32, aa.BF16, aa.F16], ids=NAMES.get)
@pytest.mark.parametrize("size", SIZES, ids=lambda s: f"t{s[0]}i{s[1]}o{s[2]}p{s[3]}")
@pytest.mark.parametrize("act", [aa.SILU, aa.GELU], ids=["silu", "gelu"])
def test_gated(size, ty, act):
    n, i, o, spare = size
    gen = np.random.default_rng(n + 3 * i + o)
    # Products of a few units: scales for activations of up to about 30 and codes of about 74.
    scale = [(np.exp(0.3 * gen.standard_normal(o)) / (100 * np.sqrt(i))).astype(np.float32) for _ in range(2)]
    w, up = Weights(gen, i, o, scale=scale[0], spare=spare), Weights(gen, i, o, scale=scale[1], spare=spare)
    x = _rows(gen, n, i, ty, spare)
    h = _host(x)
    _check_gated(ty, _product(w, ty, x, spare, up, act), plain.product8(h, w.codes, w.scale),
                 plain.product8(h, up.codes, up.scale), act)


@pytest.mark.parametrize("act", [aa.SILU, aa.GELU], ids=["silu", "gelu"])
def test_gate_over_its_whole_range(act):
    """One input, so that the gate runs over -300 to 300 and past the range of e^x."""
    gen = np.random.default_rng(1)
    g = np.concatenate([np.linspace(-300, 300, 999), [0.0]]).astype(np.float32)
    w = Weights(gen, 1, 1000, codes=np.full((1000, 1), 1, np.int8), scale=g)
    up = Weights(gen, 1, 1000, codes=np.full((1000, 1), 1, np.int8), scale=np.full(1000, 0.5, np.float32))
    x = _dev(np.ones((1, 1), np.float32))
    h = plain.product8(np.ones((1, 1)), w.codes, w.scale)
    _check_gated(aa.F32, _product(w, aa.F32, x, 0, up, act), h, plain.product8(np.ones((1, 1)), up.codes, up.scale), act)


def _codes_of(x, n_pad):
    """The codes and scales that the library finds, through rows that pick one input each."""
    gen = np.random.default_rng(0)
    torch = torch_cuda()
    n, i = x.shape
    w = Weights(gen, i, i, codes=np.eye(i, dtype=np.int8), scale=np.ones(i, np.float32))
    xx = torch.cat([x, x[:1].expand(n_pad, i)]) if n_pad else x
    return _host(_product(w, aa.F32, xx.contiguous()))[:n]


@pytest.mark.parametrize("n_pad", [0, 100, 600], ids=["few", "some", "many"])
def test_codes_next_to_borders(n_pad):
    """Ties go to even codes; the numbers next to a tie go their own way, at scales that are no powers of two too."""
    halves = np.arange(-126.5, 127, 1.0)
    rows = []
    for top in (127.0, 127.0 * 2.0 ** -90, 254.0 * 2.0 ** 100, 100.1, 3.3e-5, 77.7):
        s = np.float64(np.float32(np.float32(top) / np.float32(127)))
        near = (halves * s).astype(np.float32)
        both = np.concatenate([near, np.nextafter(near, np.float32(np.inf)), np.nextafter(near, np.float32(-np.inf))])
        rows.append(np.concatenate([[np.float32(top), -np.float32(top)], both]))
    x = np.stack(rows).astype(np.float32)
    s, c = plain.quantise8(x)
    # One f32 product of a code and a scale each.
    assert np.array_equal(_codes_of(_dev(x), n_pad), s.astype(np.float32)[:, None] * c.astype(np.float32))


@pytest.mark.parametrize("n_pad", [0, 100, 600], ids=["few", "some", "many"])
def test_rows_of_zeros_tiny_huge_and_not_finite(n_pad):
    gen = np.random.default_rng(8)
    x = gen.standard_normal((9, 200)).astype(np.float32)
    x[0] = 0
    x[1] *= 1e-35               # below 2^-100: zeros
    x[2] *= 1e-29               # above it
    x[3] = x[3] / np.abs(x[3]).max() * np.float32(3.4e38)
    x[4, 7], x[5, 199], x[6, 0] = np.nan, np.inf, -np.inf
    x[7] = -0.0
    scale = np.array([1.0, 1e-38, 1e-44, 1e30, 0.0, -1.0, np.nan, np.inf], np.float32)
    w = Weights(gen, 200, 8, scale=scale)
    pad = np.repeat(x[8:], n_pad, 0)
    got = _host(_product(w, aa.F32, _dev(np.concatenate([x, pad]))))[:9]
    with np.errstate(all="ignore"):
        want = plain.product8(x, w.codes, scale)
    assert np.isnan(got[4:7]).all() and np.isnan(got[:, 6]).all() and (got[[0, 1, 7]][:, :6] == 0).all()
    for r in (2, 3, 8):
        big = np.abs(want[r, :6]) > 3.4e38 * 1.001
        assert np.array_equal(got[r, :6][big], np.sign(want[r, :6][big]) * np.inf)
        ok = np.abs(want[r, :6]) < 3.4e38
        assert np.all(np.abs(got[r, :6] - want[r, :6])[ok] <= (3.01 * U * np.abs(want[r, :6]) + 2.0 ** -149)[ok])


def test_longest_rows_and_extreme_codes():
    gen = np.random.default_rng(3)
    i = 131072
    codes = np.stack([np.full(i, -128), np.full(i, 127), np.where(np.arange(i) % 2, 127, -128)]).astype(np.int8)
    w = Weights(gen, i, 3, codes=codes, scale=np.ones(3, np.float32))
    for n in (1, 2, 130):
        x = np.ones((n, i), np.float32)
        x[-1, ::3] = -1
        _check(aa.F32, _product(w, aa.F32, _dev(x)), plain.product8(x, codes, w.scale))


def test_a_rows_bits_do_not_depend_on_the_batch():
    gen = np.random.default_rng(4)
    w, up = Weights(gen, 700, 300), Weights(gen, 700, 300)
    x = _rows(gen, 700, 700, aa.F32, 0)
    for u in (None, up):
        whole = _product(w, aa.F32, x, up=u)
        for n in (1, 2, 16, 30, 60, 128, 129, 512):
            assert (_product(w, aa.F32, x[:n], up=u) == whole[:n]).all(), n


@pytest.mark.parametrize("kind", [-1] + list(aa.KINDS), ids=lambda k: "f32" if k < 0 else aa.KIND_NAMES[k])
@pytest.mark.parametrize("shape", [(256, 1), (512, 50), (4096, 33)], ids=str)
def test_convert_and_unpack(kind, shape):
    torch = torch_cuda()
    i, o = shape
    gen = synth.rng(i + o + kind)
    dev = aa.DeviceOps()
    if kind < 0:
        w = gen.standard_normal((o, i)).astype(np.float32)
        w[0] = 0
        values = w
    else:
        w = synth.weight_np(kind, o, i, gen)
        values = oracle.dequant(kind, w, i, o).reshape(o, i)
    p = torch.full((dev.w8_bytes(i, o),), 0x81, dtype=torch.uint8, device="cuda")
    d, out = _dev(w), torch.full((o, i), 7.0, device="cuda")
    dev.w8_convert(kind, d.data_ptr(), i, o, p.data_ptr(), stream())
    dev.w8_unpack(p.data_ptr(), i, o, out.data_ptr(), stream())
    sync()
    s, c = plain.quantise8(values)
    assert np.array_equal(out.cpu().numpy(), s.astype(np.float32)[:, None] * c.astype(np.float32))
    x = gen.standard_normal((3, i)).astype(np.float32)
    y = torch.empty(3, o, device="cuda")
    work = torch.empty(dev.w8_work_bytes(3, i), dtype=torch.uint8, device="cuda")
    dx = _dev(x)
    dev.w8_matmul(p.data_ptr(), i, o, aa.F32, dx.data_ptr(), i, 3, y.data_ptr(), o, work.data_ptr(), stream())
    sync()
    _check(aa.F32, y, plain.product8(x, c, s.astype(np.float32)))


def test_convert_of_odd_f32_rows_and_rows_that_are_not_finite():
    torch = torch_cuda()
    gen = np.random.default_rng(6)
    w = gen.standard_normal((19, 77)).astype(np.float32)
    w[3, 5], w[4, 76] = np.nan, np.inf
    w[18] *= 1e-33
    dev = aa.DeviceOps()
    p = torch.empty(dev.w8_bytes(77, 19), dtype=torch.uint8, device="cuda")
    d, out = _dev(w), torch.empty(19, 77, device="cuda")
    dev.w8_convert(-1, d.data_ptr(), 77, 19, p.data_ptr(), stream())
    dev.w8_unpack(p.data_ptr(), 77, 19, out.data_ptr(), stream())
    sync()
    s, c = plain.quantise8(w)
    assert np.array_equal(out.cpu().numpy(), s.astype(np.float32)[:, None] * c.astype(np.float32), equal_nan=True)
    assert np.isnan(s[3:5]).all() and s[18] == 0


@pytest.mark.parametrize("n", [1, 9, 60, 130, 600])
def test_captured_into_a_graph_and_on_two_streams(n):
    """Replays with other inputs and eager work between them, and calls with a
    workspace each on two streams: the eager results."""
    torch = torch_cuda()
    gen = np.random.default_rng(n)
    w, up = Weights(gen, 1000, 200), Weights(gen, 1000, 200)
    xs = [_rows(gen, n, 1000, aa.BF16, 0) for _ in range(4)]
    want = [(_product(w, aa.BF16, x).clone(), _product(w, aa.BF16, x, up=up).clone()) for x in xs]
    x, y, z = xs[0].clone(), torch.empty_like(want[0][0]), torch.empty_like(want[0][0])
    work = w.work(n)

    def call(x, y, z, work, sp):
        w.dev.w8_matmul(w.p.data_ptr(), 1000, 200, aa.BF16, x.data_ptr(), 1000, n, y.data_ptr(), 200, work.data_ptr(), sp)
        w.dev.w8_gated(w.p.data_ptr(), up.p.data_ptr(), 1000, 200, 0, aa.BF16, x.data_ptr(), 1000, n, z.data_ptr(), 200,
                       work.data_ptr(), sp)
    side = torch.cuda.Stream()
    sync()
    with torch.cuda.stream(side):
        call(x, y, z, work, side.cuda_stream)
    sync()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        call(x, y, z, work, torch.cuda.current_stream().cuda_stream)
    for x2, (a, b) in zip(xs, want):
        x.copy_(x2)
        y.fill_(0)
        graph.replay()
        torch.ones(1000, device="cuda").sum()
        sync()
        assert torch.equal(y, a) and torch.equal(z, b)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[(torch.empty_like(y), torch.empty_like(z)) for _ in range(10)] for _ in streams]
    works = [w.work(n) for _ in streams]
    sync()
    for k in range(10):
        for s, o, wk, x2 in zip(streams, outs, works, xs):
            call(x2, *o[k], wk, s.cuda_stream)
    sync()
    for o, (a, b) in zip(outs, want):
        for c, d in o:
            assert torch.equal(c, a) and torch.equal(d, b)


@pytest.mark.parametrize("ty", [aa.F32, aa.BF16, aa.F16], ids=NAMES.get)
@pytest.mark.parametrize("size", [(3, 4097, 20, 0), (60, 5003, 33, 1), (256, 4111, 17, 0), (257, 4111, 17, 0),
                                  (7, 16385, 40, 3), (33, 40007, 5, 0)], ids=lambda s: f"t{s[0]}i{s[1]}o{s[2]}p{s[3]}")
def test_odd_wide_rows_of_few_tokens(size, ty):
    test_product(size, ty)
