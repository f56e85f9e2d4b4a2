"""The 4-bit cache calls at the edges of what their contracts allow."""
import numpy as np
import pytest

import aspida_amd as aa
import kv4_plain as plain
from gpu_helpers import stream, sync, torch_cuda
from test_gpu_kv4 import HALF, NAMES, Cache, _attend, _check, _dev, _filled, _host, _i32, _starts, _t

pytestmark = pytest.mark.gpu


def test_evict_shrinks_lengths_in_place():
    """new_len may be kv_len: every kv head still selects from the old length."""
    torch = torch_cuda()
    gen = np.random.default_rng(17)
    dim, kv, keep = 64, 8, 70
    lens = [int(n) for n in gen.integers(1, 700, 24)] + [0, 70, 71]
    c = _filled(gen, dim, kv, lens)
    acc = _dev(gen.random((len(lens), kv, 700)).astype(np.float32))
    results = []
    for in_place in (False, True):
        dst = Cache(np.random.default_rng(1), dim, kv, len(lens), 2, spare=0, fill=0)
        ln = _i32(lens)
        new_len = ln if in_place else _i32([99] * len(lens))
        idx, out = _i32(np.full((len(lens), kv, keep), 99)), torch.full((len(lens), kv, keep), 7.0, device="cuda")
        c.dev.kv4_evict(c.c, len(lens), ln.data_ptr(), acc.data_ptr(), 700, keep, 3, 20, dst.c, new_len.data_ptr(),
                        idx.data_ptr(), out.data_ptr(), stream())
        sync()
        assert new_len.cpu().tolist() == [min(n, keep) for n in lens]
        results.append((idx, out, dst.pages))
    for a, b in zip(*results):
        assert torch.equal(a, b)


@pytest.mark.parametrize("window", [0, 3])
@pytest.mark.parametrize("rows,heads", [(10, 4), (40, 1), (20, 8)])
def test_slot_weights_past_max_rows_are_nan_in_every_slot_seen(rows, heads, window):
    """Also in slots that only rows past the first 16 columns see, and in no others."""
    torch = torch_cuda()
    gen = np.random.default_rng(3)
    lens = [100, 80]
    c = _filled(gen, 128, 1, lens)
    q = _dev(gen.standard_normal((rows + 1, heads * 128)).astype(np.float32))
    st = [0, rows, rows + 1]
    _, lse = _attend(c, aa.F32, q, st, lens, heads, 0.1, window)
    base = gen.random((2, 1, 128)).astype(np.float32)
    a, out = _dev(base), torch.zeros(2, 1, 128, device="cuda")
    s, l = _i32(st), _i32(lens)
    for max_rows in (1, rows - 1):
        c.dev.kv4_weigh(c.c, aa.F32, q.data_ptr(), heads * 128, heads, rows + 1, 2, s.data_ptr(), max_rows, l.data_ptr(),
                        0.1, lse.data_ptr(), a.data_ptr(), out.data_ptr(), 128, stream(), window=window)
        sync()
        o, lo = _host(out)[:, 0], max(0, 100 - rows - window + 1) if window else 0
        assert np.isnan(o[0, lo:100]).all() and np.isfinite(o[1]).all()
        assert np.array_equal(o[0, :lo], base[0, 0, :lo]) and np.array_equal(o[0, 100:], base[0, 0, 100:])


@pytest.mark.parametrize("rows,many", [([5, 4], False), ([100, 90], True)], ids=["few", "many"])
def test_windows_beyond_every_slot_hide_nothing(rows, many):
    """Up to INT_MAX, also for a sequence with rows below slot 0."""
    torch = torch_cuda()
    gen = np.random.default_rng(13)
    dim, heads, kv, lens = 128, 4, 2, [rows[0] - 3, 300]
    c = _filled(gen, dim, kv, lens, max_pages=5)
    st = _starts(rows)
    q = _dev(gen.standard_normal((st[-1], heads * dim)).astype(np.float32))
    want, wl = _attend(c, aa.F32, q, st, lens, heads, 0.1, many=many)
    assert np.isfinite(_host(want)).all() and (wl[3:] > -100).all()
    s, l = _i32(st), _i32(lens)
    weights = []
    for window in (0, 5 * 64, 1 << 30, 2 ** 31 - 1):
        out, lse = _attend(c, aa.F32, q, st, lens, heads, 0.1, window, many=many)
        assert (out == want).all() and (lse == wl).all()
        a = torch.zeros(2, kv, 320, device="cuda")
        c.dev.kv4_weigh(c.c, aa.F32, q.data_ptr(), heads * dim, heads, int(st[-1]), 2, s.data_ptr(), max(rows),
                        l.data_ptr(), 0.1, lse.data_ptr(), 0, a.data_ptr(), 320, stream(), window=window)
        sync()
        weights.append(a)
    assert all((w == weights[0]).all() for w in weights)


@pytest.mark.parametrize("dim,heads,kv,rows,lens", [
    (64, 4, 1, [1], [9001]), (64, 64, 8, [1] * 70, [(131 * i) % 900 for i in range(70)]), (128, 64, 8, [1] * 63 + [9], [400] * 64),
    (128, 4, 1, [1] * 5 + [40], [3000] * 6), (256, 8, 8, [1, 1, 1], [2500, 1, 700]), (256, 2, 1, [7] * 9, [333] * 9),
], ids=lambda v: str(v) if isinstance(v, int) else f"{len(v)}x{max(v)}")
def test_attention_stays_in_its_workspace(dim, heads, kv, rows, lens):
    """One workspace for calls of all shapes, with memory behind it that must
    stay; what calls before left in it does not matter."""
    torch = torch_cuda()
    gen = np.random.default_rng(dim + len(rows))
    c = _filled(gen, dim, kv, lens)
    st, n = _starts(rows), sum(rows)
    q = _dev(2 * gen.standard_normal((n, heads * dim)).astype(np.float32))
    s, l = _i32(st), _i32(lens)
    size = c.dev.kv4_attention_work_bytes(c.c, kv, 1, 1, 1)
    outs = []
    for fill in (0xFF, 0x3C):
        work = torch.full((size + 65536,), fill, dtype=torch.uint8, device="cuda")
        out, lse = torch.full((n, heads * dim), 7.0, device="cuda"), torch.full((n, heads), 7.0, device="cuda")
        c.dev.kv4_attention(c.c, aa.F32, q.data_ptr(), heads * dim, heads, n, len(lens), s.data_ptr(), max(rows),
                            l.data_ptr(), dim ** -0.5, out.data_ptr(), heads * dim, work.data_ptr(), stream(),
                            lse=lse.data_ptr())
        sync()
        assert (work[size:] == fill).all()
        outs.append((out, lse))
    _check(c, aa.F32, q, st, lens, heads, dim ** -0.5, 0, *outs[0])
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])


@pytest.mark.parametrize("rows,heads,kv,ty", [(131073, 128, 1, aa.BF16), (79, 16384, 16384, aa.F32), (5, 65535, 65535, aa.F16)],
                         ids=["one_kv_head", "kv_heads", "few_rows"])
def test_attention_of_more_columns_than_a_launch_of_column_tiles(rows, heads, kv, ty):
    """Every row of millions of columns is written: with a window of one slot
    each is the value at its own slot."""
    torch = torch_cuda()
    dim, pages = 64, -(-rows // 64)
    c = Cache(np.random.default_rng(1), dim, kv, 1, pages, spare=0, fill=0)
    gen = torch.Generator(device="cuda").manual_seed(5)
    k, v = (torch.randn(rows, kv, dim, device="cuda", generator=gen) for _ in range(2))
    c.append(aa.F32, k, v, [0, rows], [rows])
    s, l = _i32([0, rows]), _i32([rows])
    c.dev.kv4_read(c.c, aa.F32, rows, 1, s.data_ptr(), l.data_ptr(), k.data_ptr(), kv * dim, v.data_ptr(), kv * dim, stream())
    q = torch.randn(rows, heads, dim, device="cuda", generator=gen, dtype=_t(ty))
    out, lse = torch.full_like(q, 777.0), torch.full((rows, heads), 777.0, device="cuda")
    work = torch.empty(c.dev.kv4_attention_work_bytes(c.c, heads, rows, 1, rows), dtype=torch.uint8, device="cuda")
    c.dev.kv4_attention(c.c, ty, q.data_ptr(), heads * dim, heads, rows, 1, s.data_ptr(), rows, l.data_ptr(), 0.125,
                        out.data_ptr(), heads * dim, work.data_ptr(), stream(), window=1, lse=lse.data_ptr())
    sync()
    for a in range(0, rows, 8192):
        b = min(rows, a + 8192)
        want = v[a:b].repeat_interleave(heads // kv, 1)
        # One weight of 1: both its f16 numbers, and the code's and the
        # minimum's part of at most 16 each, a few roundings of 2^-22.
        assert ((out[a:b].float() - want).abs() <= HALF[ty] * want.abs() * (1 + 2.0 ** -10) + 2.0 ** -16).all()
        score = (q[a:b].float() * k[a:b].repeat_interleave(heads // kv, 1)).sum(-1) * 0.125
        assert ((lse[a:b] - score).abs() <= 2.0 ** -14).all()
    del c, k, v, q, out, lse
    torch.cuda.empty_cache()


@pytest.mark.parametrize("rows,many", [(3, False), (90, True)], ids=["few", "many"])
@pytest.mark.parametrize("bits", [10, 18, 22, 24, 26, 28, 30])
@pytest.mark.parametrize("ty", [aa.F32, aa.BF16], ids=NAMES.get)
def test_attention_of_scores_of_any_size(ty, bits, rows, many):
    """Scores around +-2^bits, where f32 holds fewer and fewer of the steps
    between them: values that are all alike come out whatever the weights."""
    gen = np.random.default_rng(bits)
    dim, heads, kv, n = 64, 4, 1, 700
    k = np.zeros((n, kv, dim), np.float32)
    k[..., :32] = 1024.0                                           # a constant group, times 32 equal queries
    k[..., 32:] = np.sort(gen.integers(0, 16, (n, 1, 1)), 0)       # steps of 1 between the slots' scores
    k[..., 32], k[..., 33] = 0, 15
    v = np.repeat(gen.standard_normal((1, kv, dim)), n, 0).astype(np.float32)
    c = Cache(gen, dim, kv, 1, 11)
    c.append(aa.F32, _dev(k), _dev(v), [0, n], [n])
    value = c.all([n])[0][1][0, 0]
    for sign in (1, -1):
        q = np.zeros((rows, heads, dim), np.float32)
        q[..., :32] = sign * 2.0 ** (bits - 15)
        q[..., 34] = 1
        out, lse = _attend(c, ty, _dev(q.reshape(rows, -1), ty), [0, rows], [n], heads, 1.0, many=many)
        off = np.abs(_host(out).reshape(-1, dim) - value)
        # One value times the sum of all weights over the same sum.
        assert np.all(off <= HALF[ty] * np.abs(value) * (1 + 2.0 ** -10) + 2.0 ** -16)
        # Between the largest score and that of all slots: 15 + log 700; sums of 2^bits in f32.
        assert np.all(np.abs(_host(lse) - sign * 2.0 ** bits) <= 22 + 2.0 ** (bits - 19))


@pytest.mark.parametrize("factor", [1.0, 2.0 ** -10, 2.0 ** -19])
def test_rope_at_the_largest_angles(factor):
    """Positions up to the ends of int, angles up to 2^50."""
    torch = torch_cuda()
    gen = np.random.default_rng(8)
    pos = np.concatenate([[-2 ** 31, 2 ** 31 - 1, -1, 0, 1], gen.integers(-2 ** 31, 2 ** 31, 1000)])
    rope = aa.Rope(8, base=3.0, scaling="linear", factor=factor)
    f, mag = rope.table()
    x = gen.standard_normal((len(pos), 1, 8)).astype(np.float32)
    dx, dp = _dev(x), _i32(pos)
    y = torch.empty_like(dx)
    aa.DeviceOps().rope(rope, aa.F32, dx.data_ptr(), 8, len(pos), 1, 8, dp.data_ptr(), y.data_ptr(), 8, stream())
    sync()
    want = plain.rotate(x, pos, f, mag, False)
    # cos, sin, two products and the result round by half a step of f32 each.
    size = np.tile(np.abs(x[..., :4]) + np.abs(x[..., 4:]), 2)
    assert np.all(np.abs(_host(y) - want) <= 4 * HALF[aa.F32] * size + HALF[aa.F32] * np.abs(want))


def test_a_prompt_with_weights_and_eviction_captured():
    """A prompt's chunks (rows behind what is cached), slot weights and an
    eviction in one graph: replays read lengths, rows and positions anew and
    give the bits of eager calls, with eager work between them."""
    torch = torch_cuda()
    gen = np.random.default_rng(23)
    dim, heads, kv, n, keep = 128, 16, 2, 700, 200
    rope = aa.Rope(dim, base=10000.0)
    src, dst = (Cache(np.random.default_rng(i), dim, kv, 2, p, spare=0, fill=0) for i, p in ((1, 40), (2, 4)))
    dev, empty = src.dev, lambda *s: torch.empty(*s, device="cuda")  # noqa: E731
    k, v, q = empty(n, kv, dim), empty(n, kv, dim), empty(n, heads, dim)
    turned, out, lse = torch.empty_like(q), torch.empty_like(q), empty(n, heads)
    acc, kept, idx = empty(2, kv, 2560), empty(2, kv, keep), torch.empty(2, kv, keep, dtype=torch.int32, device="cuda")
    starts, lens, new, pos = _i32([0, 1, n]), _i32([0, 0]), _i32([0, 0]), _i32(np.zeros(n))
    work = torch.empty(dev.kv4_attention_work_bytes(src.c, heads, n, 2, n), dtype=torch.uint8, device="cuda")
    few = torch.empty_like(out)

    def run():
        sp, row = stream(), kv * dim
        dev.kv4_append(src.c, aa.F32, k.data_ptr(), row, v.data_ptr(), row, n, 2, starts.data_ptr(), lens.data_ptr(), rope,
                       pos.data_ptr(), sp)
        dev.rope(rope, aa.F32, q.data_ptr(), heads * dim, n, heads, dim, pos.data_ptr(), turned.data_ptr(), heads * dim, sp)
        for rows, o in ((n, out), (8, few)):  # the kernel of many rows, and that of few (rows past 8 are NaN)
            m = n if rows == n else 12
            dev.kv4_attention(src.c, aa.F32, turned.data_ptr(), heads * dim, heads, m, 2, starts.data_ptr(), rows,
                              lens.data_ptr(), dim ** -0.5, o.data_ptr(), heads * dim, work.data_ptr(), sp,
                              lse=lse.data_ptr() if rows == n else 0)
        dev.kv4_weigh(src.c, aa.F32, turned.data_ptr(), heads * dim, heads, n, 2, starts.data_ptr(), n, lens.data_ptr(),
                      dim ** -0.5, lse.data_ptr(), 0, acc.data_ptr(), 2560, sp)
        dev.kv4_evict(src.c, 2, lens.data_ptr(), acc.data_ptr(), 2560, keep, 4, 32, dst.c, new.data_ptr(), idx.data_ptr(),
                      kept.data_ptr(), sp)

    def turns(call):
        got = []
        for i, (split, before) in enumerate(((1, (0, 0)), (350, (1, 699)), (650, (351, 1049)))):
            g = torch.Generator(device="cuda").manual_seed(i)
            for x in (k, v, q):
                x.copy_(torch.randn(x.shape, device="cuda", generator=g))
            starts.copy_(_i32([0, split, n]))
            lens.copy_(_i32([before[0] + split, before[1] + n - split]))
            pos.copy_(torch.cat([torch.arange(split, device="cuda") + before[0],
                                 torch.arange(n - split, device="cuda") + before[1]]).int())
            few.zero_()
            call()
            sync()
            assert torch.isfinite(out).all() and new.cpu().tolist() == [min(int(m), keep) for m in lens.cpu()]
            got.append([x.clone() for x in (out, lse, few, acc, idx, kept, dst.pages)])
        return got
    eager = turns(run)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        run()
    sync()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        run()

    def replay():
        graph.replay()
        torch.ones(1000, device="cuda").sum()
    for _ in range(2):
        src.pages.zero_(), dst.pages.zero_()
        for a, b in zip(eager, turns(replay)):
            for x, y in zip(a, b):
                assert torch.equal(x.nan_to_num(123.0) if x.is_floating_point() else x,
                                   y.nan_to_num(123.0) if y.is_floating_point() else y)
