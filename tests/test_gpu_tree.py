"""Trees of drafted tokens on the GPU: masks, attention, the greedy choice and
the kept slots, against plain forms in 64 bits and whole numbers.

Attention's bounds are those that test_gpu_kv4.py derives for f32 activations,
for every type: softmax weights are two f16 numbers for all of them, and 16-bit
queries are exact.  u = 2^-24: scores S = 2^-19 of scale sum |q| (|d code| +
|m|), weights 2 S + 2^-20 + (n / 16 + 64) u, the result h_T more of itself.
"""
import numpy as np
import pytest

import aspida_amd as aa
import kv4_plain
import more_plain as plain
from gpu_helpers import stream, sync, torch_cuda
from test_gpu_kv4 import (HALF, NAMES, TINY, U, Cache, _attend, _dev, _filled, _host, _i32, _kv, _starts, _t)

pytestmark = pytest.mark.gpu


def _forest(gen, n, roots=False):
    """Parents of n rows; with roots, some rows name no earlier row."""
    p = np.array([-1] + [int(gen.integers(max(0, i - 6), i)) for i in range(1, n)], np.int32)[:n]
    if roots and n > 2:
        for i in gen.choice(np.arange(1, n), max(1, n // 8), replace=False):
            p[i] = gen.choice([-1, -7, i, i + 1, 1 << 30])
    return p


# ---- masks and positions -------------------------------------------------------

@pytest.mark.parametrize("rows,words", [([1], 1), ([8], 1), ([31, 32, 33, 0, 64], 3), ([60], 2), ([100, 7], 1),
                                        ([1000], 32), ([4096], 128), ([4100, 2], 128)], ids=str)
def test_masks_and_positions(rows, words):
    torch = torch_cuda()
    gen = np.random.default_rng(sum(rows))
    starts, n = _starts(rows), sum(rows)
    trees = [_forest(gen, r, True) for r in rows]
    lens = [r + 100 * i for i, r in enumerate(rows)]
    if len(rows) > 1:
        lens[-1] = 1  # rows below slot 0 keep their places in the tree
    parent, st, ln = _i32(np.concatenate(trees)), _i32(starts), _i32(lens)
    pos = torch.full((n + 3,), 7, dtype=torch.int32, device="cuda")
    mask = torch.full((n + 3, words), 7, dtype=torch.int32, device="cuda")
    dev = aa.DeviceOps()
    dev.tree(parent.data_ptr(), n + 3, len(rows), st.data_ptr(), ln.data_ptr(), pos.data_ptr(), mask.data_ptr(), words,
             stream())
    sync()
    got_p, got_m = pos.cpu().numpy(), mask.cpu().numpy().view(np.uint32)
    assert (got_p[n:] == 7).all() and (got_m[n:] == 7).all()
    for b, r in enumerate(rows):
        on = plain.ancestors(trees[b])
        depth = on.sum(1) - 1
        if r > 4096:  # rows past that belong to no tree
            on[4096:], depth[4096:] = False, 0
        a = starts[b]
        assert np.array_equal(got_m[a:a + r], plain.mask_words(on, words))
        assert np.array_equal(got_p[a:a + r], lens[b] - r + depth)
    # Either alone.
    p2, m2 = torch.zeros_like(pos), torch.zeros_like(mask)
    dev.tree(parent.data_ptr(), n, len(rows), st.data_ptr(), ln.data_ptr(), p2.data_ptr(), stream=stream())
    dev.tree(parent.data_ptr(), n, len(rows), st.data_ptr(), ln.data_ptr(), 0, m2.data_ptr(), words, stream())
    sync()
    assert torch.equal(p2[:n], pos[:n]) and torch.equal(m2[:n], mask[:n])


# ---- attention -------------------------------------------------------------------

def _tree_attend(c, ty, q, starts, lens, heads, scale, mask, words, window=0, max_rows=None, want_lse=True,
                 out_stride=None, n=None):
    torch = torch_cuda()
    n = q.shape[0] if n is None else n
    st, ln = _i32(starts), _i32(lens)
    stride = out_stride or heads * c.dim
    out = torch.full((q.shape[0], stride), 7.0, dtype=_t(ty), device="cuda")
    lse = torch.full((q.shape[0], heads), 7.0, device="cuda")
    mr = max_rows or max(1, int(np.diff(starts).max()))
    work = torch.full((c.dev.kv4_tree_attention_work_bytes(c.c, heads, n, len(lens), mr),), 0xFF, dtype=torch.uint8,
                      device="cuda")
    c.dev.kv4_tree_attention(c.c, ty, q.data_ptr(), q.stride(0), heads, n, len(lens), st.data_ptr(), mr, ln.data_ptr(),
                             mask.data_ptr(), words, scale, out.data_ptr(), stride, work.data_ptr(), stream(),
                             window=window, lse=lse.data_ptr() if want_lse else 0)
    sync()
    return out, lse


def _check_tree(c, ty, q, starts, lens, heads, scale, ons, window, out, lse, kvs=None):
    kvs = kvs or c.all(lens)
    hq = _host(q)[:, :heads * c.dim].reshape(-1, heads, c.dim)
    ho, hl = _host(out)[:, :heads * c.dim].reshape(-1, heads, c.dim), _host(lse)
    for b, n in enumerate(lens):
        r0, r1 = starts[b], starts[b + 1]
        if r0 == r1:
            continue
        see = plain.tree_sees(ons[b], n - (r1 - r0), window)
        k, v = kvs[b]
        want, wl, pv, sk = plain.attend(hq[r0:r1], k, v, scale, see)
        s, sums = 2.0 ** -19 * sk, (n / 16 + 64) * U
        bo = (2 * s + 2.0 ** -20 + sums)[..., None] * pv + HALF[ty] * np.abs(want) + TINY[ty]
        eo = np.abs(ho[r0:r1] - want)
        assert np.all(eo <= bo), (b, np.max(eo / bo))
        with np.errstate(invalid="ignore"):
            bl = s + 2.0 ** -20 + sums + U * np.abs(wl)
            el = np.where(wl == hl[r0:r1], 0, np.abs(hl[r0:r1] - wl))
            assert np.all(el <= np.where(np.isfinite(bl), bl, 0)), (b, np.nanmax(el / bl))


TREES = [
    # dim, heads, kv, rows, lens, window
    (128, 4, 1, [1], [1], 0),
    (128, 32, 8, [8], [777], 0),
    (128, 32, 8, [1, 1, 1, 1], [17, 1, 64, 65], 0),
    (128, 8, 2, [5, 9, 1, 26], [5, 40, 300, 1000], 0),      # one that is all tree
    (128, 8, 8, [3, 17], [31, 300], 0),                     # a query head per kv head
    (128, 5, 1, [7, 2], [129, 33], 0),                      # an odd group
    (128, 64, 8, [60], [2000], 0),
    (128, 40, 1, [4, 13], [100, 700], 0),                   # more heads than a tile
    (64, 6, 3, [12, 33], [63, 500], 0),
    (64, 24, 1, [2, 40], [5, 200], 0),
    (256, 8, 4, [6, 19], [16, 400], 0),
    (256, 2, 1, [3], [3], 0),
    (256, 16, 2, [50], [333], 0),
    (128, 8, 2, [5, 9], [90, 700], 1),                      # itself alone, or less
    (128, 8, 2, [12, 30], [200, 700], 8),                   # trees deeper than the window
    (128, 8, 2, [12, 30], [700, 90], 64),
    (64, 8, 2, [100], [1000], 300),
    (128, 8, 2, [5, 0, 4], [3, 10, 0], 0),                  # rows below slot 0, none, an empty sequence
    (128, 8, 2, [5, 6], [3, 2], 3),
    (128, 4, 2, [130], [130], 0),                           # wide masks, all tree
    (128, 16, 2, [64, 65, 63, 128], [64 * 3, 64 * 5 + 1, 64 * 2, 1000], 0),
    (128, 8, 2, [300], [3000], 0),
    (64, 2, 1, [3] * 70, list(range(3, 73)), 0),            # more sequences than a wave has lanes
]


@pytest.mark.parametrize("ty", [aa.F32, aa.BF16, aa.F16], ids=NAMES.get)
@pytest.mark.parametrize("case", TREES, ids=lambda c: f"d{c[0]}h{c[1]}k{c[2]}r{'_'.join(map(str, c[3][:4]))}n{'_'.join(map(str, c[4][:4]))}w{c[5]}")
@pytest.mark.parametrize("masks", ["tree", "any"])
def test_tree_attention(case, ty, masks):
    dim, heads, kv, rows, lens, window = case
    gen = np.random.default_rng(sum(rows) + sum(lens) + heads)
    c = _filled(gen, dim, kv, lens)
    starts = _starts(rows)
    q = _dev((2 * gen.standard_normal((sum(rows), heads * dim))).astype(np.float32), ty)
    words = max(1, -(-max(rows) // 32))
    if masks == "tree":
        ons = [plain.ancestors(_forest(gen, r)) for r in rows]
    else:  # any rows, some none at all
        ons = [gen.random((r, r)) < gen.choice([0, 0.1, 0.5, 1], (r, 1)) for r in rows]
        words += 1
    bits = [plain.mask_words(on, words) if len(on) else np.zeros((0, words), np.uint32) for on in ons]
    # Bits past a sequence's rows say nothing.
    for on, m in zip(ons, bits):
        if masks == "any" and len(on):
            m[:, -1] = 0xFFFFFFFF
    mask = _dev(np.concatenate(bits).view(np.int32))
    scale = -0.2 if masks == "any" else dim ** -0.5
    out, lse = _tree_attend(c, ty, q, starts, lens, heads, scale, mask, words, window)
    _check_tree(c, ty, q, starts, lens, heads, scale, ons, window, out, lse)


SHARES = [
    # dim, heads, kv, rows, lens, window: shares of the slots' axis and their joins
    (128, 32, 8, [30], [20000], 0),
    (128, 8, 2, [5, 1, 20, 3], [9000, 40, 3000, 12000], 0),
    (128, 64, 8, [60], [7001], 4000),
    (64, 16, 2, [16] * 8, [2000, 100, 4000, 16, 700, 1, 64, 3000], 0),
    (256, 8, 2, [9, 33], [5000, 2500], 0),
]


@pytest.mark.parametrize("ty", [aa.F32, aa.BF16], ids=NAMES.get)
@pytest.mark.parametrize("case", SHARES, ids=lambda c: f"d{c[0]}h{c[1]}k{c[2]}s{len(c[3])}n{max(c[4])}w{c[5]}")
def test_tree_attention_shares_and_parts(case, ty):
    test_tree_attention(case, ty, "tree")


def test_a_chain_is_causal_attention():
    """A tree without branches sees what rows one behind the other see."""
    gen = np.random.default_rng(2)
    rows, lens, heads = [9, 40], [300, 100], 8
    c = _filled(gen, 128, 2, lens)
    q = _dev(gen.standard_normal((49, heads * 128)).astype(np.float32))
    ons = [np.tril(np.ones((r, r), bool)) for r in rows]
    mask = _dev(np.concatenate([plain.mask_words(on, 2) for on in ons]).view(np.int32))
    for window in (0, 50):
        a, la = _tree_attend(c, aa.F32, q, _starts(rows), lens, heads, 0.1, mask, 2, window)
        b, lb = _attend(c, aa.F32, q, _starts(rows), lens, heads, 0.1, window)
        assert (a - b).abs().max() < 1e-5 and (la - lb).abs().max() < 1e-5


def test_strides_max_rows_and_untouched_memory():
    """Rows in a wider buffer from an odd element on, no lse, rows behind the last sequence, and a max_rows
    below the rows there are (NaN behind it) and above them."""
    torch = torch_cuda()
    gen = np.random.default_rng(5)
    rows, lens, heads, dim = [7, 30], [100, 400], 8, 64
    c = _filled(gen, dim, 2, lens)
    starts = _starts(rows)
    ons = [plain.ancestors(_forest(gen, r)) for r in rows]
    mask = _dev(np.concatenate([plain.mask_words(on, 1) for on in ons]).view(np.int32))
    buf = torch.zeros((37 + 2) * (heads * dim + 5) + 1, dtype=torch.bfloat16, device="cuda")
    q = buf[1:].view(39, heads * dim + 5)
    q.copy_(_dev(gen.standard_normal(q.shape).astype(np.float32)))
    for mr in (30, 900):
        out, lse = _tree_attend(c, aa.BF16, q, starts, lens, heads, 0.1, mask, 1, max_rows=mr, out_stride=heads * dim + 3,
                                n=39)
        assert (out[:, heads * dim:] == 7).all() and (out[37:] == 7).all() and (lse[37:] == 7).all()
        _check_tree(c, aa.BF16, q[:37], starts, lens, heads, 0.1, ons, 0, out[:37], lse[:37])
    o2, l2 = _tree_attend(c, aa.BF16, q, starts, lens, heads, 0.1, mask, 1, want_lse=False, n=39)
    assert torch.equal(o2[:37], out[:37, :heads * dim]) and (l2 == 7).all()
    o3, l3 = _tree_attend(c, aa.BF16, q, starts, lens, heads, 0.1, mask, 1, max_rows=10, n=39)
    assert torch.isnan(o3[17:37]).all() and torch.isnan(l3[17:37]).all()
    assert torch.equal(o3[:17], o2[:17]) and (o3[37:] == 7).all()


@pytest.mark.parametrize("group", [1, 8])
@pytest.mark.parametrize("ty", [aa.F32, aa.BF16], ids=NAMES.get)
def test_unseen_slots_never_matter_and_seen_ones_always(ty, group):
    """Rows that no mask names hold NaN bytes; a row that sees a token beyond
    the format, a page that is not there or a slot past the table is NaN, and
    no other row is."""
    torch = torch_cuda()
    gen = np.random.default_rng(11)
    dim, kv, n, r = 128, 2, 190, 20
    heads = kv * group
    c = Cache(gen, dim, kv, 1, 3)  # 192 slots
    k, v = _kv(gen, n, kv, dim)
    c.append(aa.F32, _dev(k[:n - 4]), _dev(v[:n - 4]), [0, n - 4], [n - 4])  # the last four are never written
    on = np.eye(r, dtype=bool)
    on[5, 2] = on[9, 7] = True
    on[16:] = False                                                     # and never seen
    q = _dev(gen.standard_normal((r, heads * dim)).astype(np.float32), ty)
    mask = lambda on: _dev(plain.mask_words(on, 1).view(np.int32))  # noqa: E731
    out, lse = _tree_attend(c, ty, q, [0, r], [n], heads, 0.1, mask(on), 1)
    kvs = [(np.concatenate([kv4_plain.stands_for(k[:n - 4]), np.zeros((4, kv, dim))]),
            np.concatenate([kv4_plain.stands_for(v[:n - 4]), np.zeros((4, kv, dim))]))]
    _check_tree(c, ty, q, [0, r], [n], heads, 0.1, [on], 0, out, lse, kvs)
    # Row 7's value is beyond the format in kv head 1: rows 7 and 9 see it.
    bad = v[n - r + 7:n - r + 8].copy()
    bad[0, 1, 3] = np.inf
    c.append(aa.F32, _dev(k[n - r + 7:n - r + 8]), _dev(bad), [0, 1], [n - r + 8])
    o2, l2 = _tree_attend(c, ty, q, [0, r], [n], heads, 0.1, mask(on), 1)
    nan = torch.isnan(o2.view(r, heads, dim)).all(-1).cpu().numpy()
    want = np.zeros((r, heads), bool)
    want[[7, 9], group:] = True
    assert np.array_equal(nan, want) and torch.equal(torch.isnan(l2).cpu(), torch.from_numpy(want))
    assert torch.equal(o2.view(r, heads, dim)[~torch.from_numpy(want)], out.view(r, heads, dim)[~torch.from_numpy(want)])
    # The tree's last page is not there: rows 0 .. 7 are at slots 170 ... in page 2 too; all see NaN but those that see none.
    t = c.host_table.copy()
    t[0, 2] = -1
    c.set_table(t)
    o3, _ = _tree_attend(c, ty, q, [0, r], [n], heads, 0.1, mask(np.zeros((r, r), bool)), 1)
    assert torch.isnan(o3).all()  # slots 128 .. 169 are before the tree
    o4, l4 = _tree_attend(c, ty, q, [0, r], [128 + r], heads, 0.1, mask(on), 1)
    assert torch.isnan(o4[:16]).all() and torch.isfinite(o4[16:].float()).all() and torch.isfinite(l4[16:]).all()
    # Slots past the table.
    c.set_table(c.host_table)
    o5, _ = _tree_attend(c, ty, q, [0, r], [192 - 16 + r], heads, 0.1, mask(np.eye(r, dtype=bool)), 1)
    assert torch.isnan(o5[16:]).all()
    o6, l6 = _tree_attend(c, ty, q, [0, r], [192 + r], heads, 0.1, mask(np.zeros((r, r), bool)), 1, window=0)
    assert o6.shape[0] == r  # sees 192 slots, all in the table
    o7, _ = _tree_attend(c, ty, q, [0, r], [193 + r], heads, 0.1, mask(np.zeros((r, r), bool)), 1)
    assert torch.isnan(o7).all()


def test_bad_row_starts_are_bounded():
    gen = np.random.default_rng(1)
    c = _filled(gen, 64, 1, [50, 60, 70])
    q = _dev(gen.standard_normal((6, 2 * 64)).astype(np.float32))
    mask = _dev(plain.mask_words(np.eye(6, dtype=bool), 1).view(np.int32))
    for starts in ([0, 100, 3, 6], [-5, 2, 1, 9], [4, 4, 4, 4]):
        out, _ = _tree_attend(c, aa.F32, q, starts, [50, 60, 70], 2, 0.1, mask, 1, max_rows=6)
        assert out.shape == (6, 128)


# ---- the greedy choice -----------------------------------------------------------

def _accept(ty, logits, rows, lens, parents, token, stride=None, alias=False):
    torch = torch_cuda()
    n, vocab = logits.shape
    starts = _starts(rows)
    dev = aa.DeviceOps()
    e = lambda m: torch.full((m + 2,), 77, dtype=torch.int32, device="cuda")  # noqa: E731
    path, count, nxt, new = e(n), e(len(rows)), e(len(rows)), e(len(rows))
    st, ln, pa, to = _i32(starts), _i32(lens), _i32(np.concatenate(parents)), _i32(token)
    work = torch.full((dev.tree_accept_work_bytes(n, vocab),), 0xFF, dtype=torch.uint8, device="cuda")
    dev.tree_accept(ty, logits.data_ptr(), stride or vocab, vocab, n, len(rows), st.data_ptr(), ln.data_ptr(),
                    pa.data_ptr(), to.data_ptr(), path.data_ptr(), count.data_ptr(), nxt.data_ptr(),
                    (ln if alias else new).data_ptr(), work.data_ptr(), stream())
    sync()
    assert (path[n:] == 77).all() and (count[len(rows):] == 77).all() and (nxt[len(rows):] == 77).all()
    return [t.cpu().numpy() for t in (path[:n], count[:-2], nxt[:-2], ln if alias else new[:-2])]


def _check_accept(got, logits, rows, lens, parents, token):
    path, count, nxt, new = got
    starts = _starts(rows)
    for b, r in enumerate(rows):
        a = starts[b]
        want, said = plain.accept(logits[a:a + r], parents[b], token[a:a + r])
        assert list(path[a:a + r]) == want + [-1] * (r - len(want)), b
        assert count[b] == len(want) and nxt[b] == said and new[b] == max(0, max(lens[b], 0) - r + len(want))


@pytest.mark.parametrize("ty", [aa.F32, aa.BF16, aa.F16], ids=NAMES.get)
@pytest.mark.parametrize("rows,vocab", [([1], 1), ([8], 7), ([8], 1000), ([5, 0, 26, 1], 32003), ([100], 257),
                                        ([2] * 90, 4096), ([40, 3], 8191), ([3000], 33), ([1, 2], 128256)], ids=str)
def test_accept(rows, vocab, ty):
    gen = np.random.default_rng(vocab + sum(rows))
    n = sum(rows)
    x = 2 * gen.standard_normal((n, vocab))
    if vocab > 4:  # equal largest ones, here and there
        x[::2, gen.integers(0, vocab, 3)] = 9.0
    x[1::7, :vocab // 2] = np.nan
    t = _dev(x.astype(np.float32), ty)
    h = _host(t)
    parents = [_forest(gen, r, True) for r in rows]
    token = gen.integers(0, vocab, n).astype(np.int32)
    for b, a in enumerate(_starts(rows)[:-1]):
        for i, p in enumerate(parents[b]):
            p = plain.tree_parent(parents[b], i)
            if p >= 0 and gen.random() < 0.7:
                token[a + i] = plain.says(h[a + p])
    lens = [r + 10 * b for b, r in enumerate(rows)]
    _check_accept(_accept(ty, t, rows, lens, parents, token, alias=len(rows) % 2 == 0), h, rows, lens, parents, token)


def test_accept_of_odd_logits():
    """Rows of NaN, of -inf, of both; infinities; zeros of both signs; odd strides; lengths below the rows."""
    torch = torch_cuda()
    x = np.zeros((8, 11), np.float32)
    x[0] = -np.inf                          # says 0
    x[1, 4] = np.inf
    x[2] = np.nan                           # says nothing
    x[3], x[3, 5] = np.nan, -np.inf         # says 5
    x[4, :] = -0.0
    x[4, 7] = 0.0                           # equal: says 0
    parents = [np.array([-1, 0, 1, 1, 0], np.int32), np.array([-1, 0], np.int32), np.array([-1], np.int32)]
    token = np.array([9, 0, 4, 4, 0, 3, 9, 1], np.int32)
    for rows_of_x in ([0, 1, 2, 3, 4, 5, 6, 7], [2, 1, 0, 3, 4, 5, 6, 7], [1, 3, 2, 0, 5, 4, 6, 7]):
        y = x[rows_of_x]
        buf = torch.full((8 * 13 + 1,), 50.0, device="cuda")[1:].view(8, 13)
        buf[:, :11] = _dev(y)
        got = _accept(aa.F32, buf[:, :11], [5, 2, 1], [5, 1, 0], parents, token, stride=13)
        _check_accept(got, y, [5, 2, 1], [5, 1, 0], parents, token)
    got = _accept(aa.F32, _dev(x[2:3]), [1], [1], [parents[2]], token[:1])
    assert list(got[0]) == [0] and got[1][0] == 1 and got[2][0] == -1


# ---- the kept slots ---------------------------------------------------------------

def _keep(c, starts, lens, path, count):
    st, ln, p, n = _i32(starts), _i32(lens), _i32(path), _i32(count)
    c.dev.kv4_keep(c.c, int(starts[-1]), len(lens), st.data_ptr(), ln.data_ptr(), p.data_ptr(), n.data_ptr(), stream())
    sync()


@pytest.mark.parametrize("dim,kv", [(64, 3), (128, 2), (256, 1)], ids=str)
@pytest.mark.parametrize("rows,lens", [([8], [8]), ([8], [70]), ([26, 5, 1], [100, 64, 7]), ([100], [190]),
                                       ([64, 64], [64 * 3, 128 + 31]), ([200, 0, 3], [450, 9, 3])], ids=str)
@pytest.mark.parametrize("paths", ["some", "all", "far", "gap"])
def test_keep(dim, kv, rows, lens, paths):
    gen = np.random.default_rng(dim + sum(rows))
    c = _filled(gen, dim, kv, lens)
    starts = _starts(rows)
    path, count = np.full(sum(rows), -1, np.int64), []
    for b, r in enumerate(rows):
        if r == 0:
            count.append(0)
            continue
        p = {"some": np.sort(gen.choice(r, max(1, r // 3), replace=False)), "all": np.arange(r),
             "far": np.array([r - 1]), "gap": np.delete(np.arange(r), r // 2) if r > 1 else np.arange(1)}[paths]
        path[starts[b]:starts[b] + len(p)] = p
        count.append(len(p))
    before = c.all(lens)
    raw = c.pages.clone()
    _keep(c, starts, lens, path, count)
    after = c.all(lens)
    for b, (r, n) in enumerate(zip(rows, lens)):
        base = n - r
        p = path[starts[b]:starts[b] + count[b]]
        for x, y in zip(before[b], after[b]):
            want = x.copy()
            want[base:base + len(p)] = x[base + p]
            assert np.array_equal(y, want), b  # what lies behind stays as it was
    if paths == "all":
        assert (raw == c.pages).all()


def test_keep_ends_at_bad_entries_and_missing_pages():
    """A path that does not ascend, or names no row, ends there; slots below 0
    and past the table are left out; a row whose page is missing reads as NaN,
    a row without a page to go to is dropped."""
    gen = np.random.default_rng(9)
    for path, good in (([0, 3, 3, 5], 2), ([1, 4, 2, 5], 2), ([2, 9, 10, 3], 2), ([-1, 0, 1, 2], 0), ([0, 2, 5, 40], 3)):
        c = _filled(gen, 64, 2, [70])
        before = c.all([70])[0]
        _keep(c, [0, 10], [70], path + [0] * 6, [4])
        for x, y in zip(before, c.all([70])[0]):
            want = x.copy()
            want[60:60 + good] = x[[60 + p for p in path[:good]]]
            assert np.array_equal(y, want), path
    c = _filled(gen, 128, 1, [70])
    before = c.all([70])[0]
    for count in (-3, 0, 99):
        _keep(c, [0, 3], [70], [0, 1, 2], [count])
    _keep(c, [0, 5], [2], [1, 2, 3, 4, -1], [4])          # rows 0 to 2 lie below slot 0: row 4's slot takes nothing
    after = c.all([70])[0]
    for x, y in zip(before, after):
        want = x.copy()
        want[0] = x[1]                                    # slot -3 + 3 takes what row 4 held
        assert np.array_equal(y, want)
    c = _filled(gen, 128, 1, [130])
    before = c.all([130])[0]
    t = c.host_table.copy()
    t[0, 1] = -1
    c.set_table(t)
    _keep(c, [0, 70], [130], [0, 1, 8, 69] + [-1] * 66, [4])  # slots 60 .. 63 take 60, 61, 68 (missing), 129
    k, v = c.read(aa.F32, [0, 64], [64])
    for x, y in zip(before, (k, v)):
        assert np.array_equal(y[:62], x[:62]) and np.isnan(y[62]).all() and np.array_equal(y[63], x[129])
    _keep(c, [0, 66], [130], list(range(1, 4)) + [-1] * 63, [3])  # to slots 64 .. 66, whose page is missing
    c.set_table(c.host_table)
    assert np.array_equal(c.all([130])[0][0][64:], before[0][64:])


def test_keep_moves_marks_of_tokens_beyond_the_format():
    gen = np.random.default_rng(13)
    c = _filled(gen, 64, 2, [40])
    k, v = _kv(gen, 4, 2, 64)
    k[3, 1, 5] = np.nan
    c.append(aa.F32, _dev(k), _dev(v), [0, 4], [40])
    _keep(c, [0, 4], [40], [0, 3, -1, -1], [2])
    got = c.all([40])[0][0]
    assert np.isnan(got[37, 1]).all() and np.isfinite(got[37, 0]).all() and np.isfinite(got[38]).all()


# ---- a step of speculative decoding --------------------------------------------------

class Decoder:
    """A decoder layer and an output head on 8-bit integer weights, over the
    4-bit cache, for any rows: as a tree, or one token after the other."""

    def __init__(self, gen, lanes, heads=8, kv=2, dim=64, hidden=256, inter=416, vocab=300, max_rows=16, max_pages=4):
        torch = torch_cuda()
        self.dev = aa.DeviceOps()
        self.sizes = heads, kv, dim, hidden, inter, vocab
        self.lanes, self.max_rows = lanes, max_rows
        self.c = Cache(gen, dim, kv, lanes, max_pages)
        self.rope = aa.Rope(dim)
        self.w = {}
        for name, o, i in (("qkv", (heads + 2 * kv) * dim, hidden), ("o", hidden, heads * dim), ("gate", inter, hidden),
                           ("up", inter, hidden), ("down", hidden, inter), ("head", vocab, hidden)):
            m = _dev((gen.standard_normal((o, i)) / np.sqrt(i)).astype(np.float32))
            p = torch.empty(self.dev.w8_bytes(i, o), dtype=torch.uint8, device="cuda")
            self.dev.w8_convert(-1, m.data_ptr(), i, o, p.data_ptr(), stream())
            sync()
            self.w[name] = p, i, o
        n = lanes * max_rows
        e = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
        i = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
        self.x, self.qkv, self.att, self.o = e(n, hidden), e(n, (heads + 2 * kv) * dim), e(n, heads * dim), e(n, hidden)
        self.h, self.y, self.logits = e(n, inter), e(n, hidden), e(n, vocab)
        self.start, self.len, self.new_len = i(lanes + 1), i(lanes), i(lanes)
        self.parent, self.token, self.pos, self.mask = i(n), i(n), i(n), i(n, 1)
        self.path, self.count, self.next = i(n), i(lanes), i(lanes)
        self.embed = _dev(gen.standard_normal((vocab, hidden)).astype(np.float32))
        self.work = torch.empty(max(self.dev.w8_work_bytes(n, max(w[1] for w in self.w.values())),
                                    self.dev.kv4_tree_attention_work_bytes(self.c.c, heads, n, lanes, max_rows),
                                    self.dev.kv4_attention_work_bytes(self.c.c, heads, n, lanes, max_rows),
                                    self.dev.tree_accept_work_bytes(n, vocab)), dtype=torch.uint8, device="cuda")

    def product(self, name, x, y, n, sp):
        p, i, o = self.w[name]
        self.dev.w8_matmul(p.data_ptr(), i, o, aa.F32, x.data_ptr(), i, n, y.data_ptr(), o, self.work.data_ptr(), sp)

    def run(self, n, tree, sp):
        heads, kv, dim, hidden, inter, vocab = self.sizes
        d, row, work = self.dev, (heads + 2 * kv) * dim, self.work.data_ptr()
        rows = self.start.data_ptr(), self.len.data_ptr()
        if tree:
            d.tree(self.parent.data_ptr(), n, self.lanes, *rows, self.pos.data_ptr(), self.mask.data_ptr(), 1, sp)
        self.product("qkv", self.x, self.qkv, n, sp)
        q = self.qkv.data_ptr()
        k, v = q + 4 * heads * dim, q + 4 * (heads + kv) * dim
        d.kv4_append(self.c.c, aa.F32, k, row, v, row, n, self.lanes, *rows, self.rope, self.pos.data_ptr(), sp)
        d.rope(self.rope, aa.F32, q, row, n, heads, dim, self.pos.data_ptr(), q, row, sp)
        if tree:
            d.kv4_tree_attention(self.c.c, aa.F32, q, row, heads, n, self.lanes, rows[0], self.max_rows, rows[1],
                                 self.mask.data_ptr(), 1, dim ** -0.5, self.att.data_ptr(), heads * dim, work, sp)
        else:
            d.kv4_attention(self.c.c, aa.F32, q, row, heads, n, self.lanes, rows[0], self.max_rows, rows[1],
                            dim ** -0.5, self.att.data_ptr(), heads * dim, work, sp)
        self.product("o", self.att, self.o, n, sp)
        (gate, i, o), (up, _, _) = self.w["gate"], self.w["up"]
        d.w8_gated(gate.data_ptr(), up.data_ptr(), i, o, aa.SILU, aa.F32, self.o.data_ptr(), i, n, self.h.data_ptr(), o,
                   work, sp)
        self.product("down", self.h, self.y, n, sp)
        self.product("head", self.y, self.logits, n, sp)
        if tree:
            d.tree_accept(aa.F32, self.logits.data_ptr(), vocab, vocab, n, self.lanes, *rows, self.parent.data_ptr(),
                          self.token.data_ptr(), self.path.data_ptr(), self.count.data_ptr(), self.next.data_ptr(),
                          self.new_len.data_ptr(), work, sp)
            d.kv4_keep(self.c.c, n, self.lanes, *rows, self.path.data_ptr(), self.count.data_ptr(), sp)


def _spec_decode(gen, dec, tokens, lens, trees, plan, run):
    """Steps of trees whose drafts follow `plan` (the tokens that decoding one
    by one gives) in part: returns each lane's tokens."""
    said = [[] for _ in lens]
    sure = list(tokens)
    for _ in range(6):
        starts, token, parent = [0], [], []
        for b in range(dec.lanes):
            t = [sure[b]]
            for i in range(1, len(trees[b])):
                depth = int(plain.ancestors(trees[b])[i].sum()) - 1
                at = len(said[b]) + depth - 1
                t.append(int(plan[b][at]) if at < len(plan[b]) and gen.random() < 0.8 else int(gen.integers(0, 300)))
            token += t
            parent += list(trees[b])
            starts.append(len(token))
        n = len(token)
        dec.start.copy_(_i32(starts))
        dec.token[:n] = _i32(token)
        dec.parent[:n] = _i32(parent)
        dec.x[:n] = dec.embed[_i32(token).long()]
        dec.len.copy_(_i32([m + len(t) for m, t in zip(lens, trees)]))
        run(n)
        sync()
        path, count, nxt, new = (t.cpu().numpy() for t in (dec.path, dec.count, dec.next, dec.new_len))
        for b in range(dec.lanes):
            rows = path[starts[b]:starts[b] + count[b]]
            assert rows[0] == 0 and new[b] == lens[b] + count[b]
            said[b] += [token[starts[b] + r] for r in rows[1:]] + [int(nxt[b])]
            sure[b], lens[b] = int(nxt[b]), int(new[b])
    return said


def _one_by_one(dec, tokens, lens, n):
    lens, toks = list(lens), list(tokens)
    said = [[] for _ in lens]
    dec.start.copy_(_i32(range(dec.lanes + 1)))
    for _ in range(n):
        dec.x[:dec.lanes] = dec.embed[_i32(toks).long()]
        lens = [m + 1 for m in lens]
        dec.len.copy_(_i32(lens))
        dec.pos[:dec.lanes] = _i32([m - 1 for m in lens])
        dec.run(dec.lanes, False, stream())
        sync()
        toks = [int(t) for t in dec.logits[:dec.lanes].argmax(1)]
        for s, t in zip(said, toks):
            s.append(t)
    return said


@pytest.mark.parametrize("captured", [False, True], ids=["eager", "captured"])
def test_speculative_decoding_gives_the_tokens_of_decoding_one_by_one(captured):
    """Trees verified step by step, with their accepted rows kept, say the
    tokens that one token a step says, and leave the same keys and values."""
    torch = torch_cuda()
    trees = [np.array([-1, 0, 1, 0, 2, 2, 1], np.int32), np.array([-1], np.int32), np.array([-1, 0, 0, 1, 3, 4], np.int32)]
    lens, tokens = [37, 1, 62], [5, 6, 7]
    dec = Decoder(np.random.default_rng(3), 3)
    ref = Decoder(np.random.default_rng(3), 3)
    fill = np.random.default_rng(4)
    kf, vf = _kv(fill, sum(lens), 2, 64)
    for d in (dec, ref):
        d.c.append(aa.F32, _dev(kf), _dev(vf), _starts(lens), lens)
    plan = _one_by_one(ref, tokens, lens, 45)
    n = sum(len(t) for t in trees)
    if captured:
        side = torch.cuda.Stream()
        keep = dec.c.pages.clone()
        sync()
        with torch.cuda.stream(side):
            dec.run(n, True, side.cuda_stream)
        sync()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            dec.run(n, True, torch.cuda.current_stream().cuda_stream)
        dec.c.pages.copy_(keep)
        run = lambda n: graph.replay()  # noqa: E731
    else:
        run = lambda n: dec.run(n, True, stream())  # noqa: E731
    now = list(lens)
    said = _spec_decode(np.random.default_rng(5), dec, tokens, now, trees, plan, run)
    assert max(len(s) for s in said) > 10  # drafts were taken
    for b in range(3):
        assert said[b] == plan[b][:len(said[b])], b
    # Keys and values: rows of both runs have the same products, but attention
    # joins other parts, so a later layer's rows may differ; this layer's may not.
    for (k, v), (k2, v2) in zip(dec.c.all(now), ref.c.all(now)):
        assert np.array_equal(k, k2) and np.array_equal(v, v2)
