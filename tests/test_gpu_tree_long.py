"""Tree attention where the page table allows many slots and the trees have
many columns, which takes the kernel that unpacks a slot once for a whole tree.
Bounds are those of test_gpu_tree.py.
"""
import numpy as np
import pytest

import aspida_amd as aa
import kv4_plain
import more_plain as plain
import test_gpu_tree as tree
from gpu_helpers import stream, torch_cuda
from test_gpu_kv4 import NAMES, Cache, _dev, _filled, _i32, _kv, _starts
from test_gpu_tree import SHARES, TREES, _check_tree, _forest, _tree_attend

pytestmark = pytest.mark.gpu
MANY = 1 << 21  # columns times slots of the table


def _widen(c, cols):
    """The same pages behind a table with entries enough."""
    pages = max(c.max_pages, MANY // cols // (64 * c.n_seq) + 1)
    t = np.full((c.n_seq, pages), -1, np.int32)
    t[:, :c.max_pages] = c.host_table
    c.max_pages, c.host_table = pages, t
    c.set_table(t)
    return c


def _cols(case):
    return max(case[3]) * case[1] // case[2]


WIDE = [c for c in TREES + SHARES if _cols(c) > 64] + [
    (128, 32, 8, [17], [777], 0),
    (128, 32, 8, [17], [17], 0),                             # all tree
    (128, 32, 8, [33, 1], [1000, 31], 0),                    # a tile and a little more
    (128, 32, 8, [40, 3, 50], [3, 2, 49], 0),                # rows below slot 0
    (128, 32, 8, [40, 3, 0, 50], [300, 90, 0, 700], 7),      # windows shorter than the trees
    (128, 32, 8, [64, 40], [3000, 64], 1000),
    (64, 32, 4, [20] * 70, list(range(20, 90)), 0),          # more sequences than a wave has lanes
    (64, 8, 2, [25], [333], 0),
    (64, 8, 2, [33, 34], [333, 4097], 65),
    (256, 16, 2, [33, 1, 0, 20], [40, 1, 0, 9000], 100),
    (256, 8, 2, [25], [333], 0),
    (128, 5, 1, [27, 2], [129, 33], 0),                      # an odd group
]


@pytest.mark.parametrize("ty", [aa.F32, aa.BF16, aa.F16], ids=NAMES.get)
@pytest.mark.parametrize("case", WIDE, ids=lambda c: f"d{c[0]}h{c[1]}k{c[2]}r{'_'.join(map(str, c[3][:4]))}n{'_'.join(map(str, c[4][:4]))}w{c[5]}")
@pytest.mark.parametrize("masks", ["tree", "any"])
def test_wide_trees(case, ty, masks, monkeypatch):
    monkeypatch.setattr(tree, "_filled", lambda *a: _widen(_filled(*a), _cols(case)))
    tree.test_tree_attention(case, ty, masks)


@pytest.mark.parametrize("ty", [aa.F32, aa.BF16], ids=NAMES.get)
def test_strides_max_rows_untouched_memory_and_the_same_bits(ty):
    torch = torch_cuda()
    gen = np.random.default_rng(5)
    rows, lens, heads, dim = [7, 50], [100, 4000], 8, 64
    c = _widen(_filled(gen, dim, 2, lens), 160)
    starts = _starts(rows)
    ons = [plain.ancestors(_forest(gen, r)) for r in rows]
    mask = _dev(np.concatenate([plain.mask_words(on, 2) for on in ons]).view(np.int32))
    buf = torch.zeros((57 + 2) * (heads * dim + 5) + 1, dtype=torch.float32 if ty == aa.F32 else torch.bfloat16, device="cuda")
    q = buf[1:].view(59, heads * dim + 5)
    q.copy_(_dev(gen.standard_normal(q.shape).astype(np.float32)))
    for mr in (50, 900):
        out, lse = _tree_attend(c, ty, q, starts, lens, heads, 0.1, mask, 2, max_rows=mr, out_stride=heads * dim + 3, n=59)
        again, _ = _tree_attend(c, ty, q, starts, lens, heads, 0.1, mask, 2, max_rows=mr, out_stride=heads * dim + 3, n=59)
        assert torch.equal(out, again)
        assert (out[:, heads * dim:] == 7).all() and (out[57:] == 7).all() and (lse[57:] == 7).all()
        _check_tree(c, ty, q[:57], starts, lens, heads, 0.1, ons, 0, out[:57], lse[:57])
    o2, l2 = _tree_attend(c, ty, q, starts, lens, heads, 0.1, mask, 2, want_lse=False, max_rows=900, n=59)
    assert torch.equal(o2[:57], out[:57, :heads * dim]) and (l2 == 7).all()
    o3, l3 = _tree_attend(c, ty, q, starts, lens, heads, 0.1, mask, 2, max_rows=40, n=59)
    assert torch.isnan(o3[47:57]).all() and torch.isnan(l3[47:57]).all()
    _check_tree(c, ty, q[:47], [0, 7, 47], [100, 3990], heads, 0.1, [ons[0], ons[1][:40, :40]], 0, o3[:47], l3[:47])
    assert (o3[57:] == 7).all()


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("ty", [aa.F32, aa.BF16], ids=NAMES.get)
def test_unseen_slots_never_matter_and_seen_ones_always(ty, dim):
    """Rows that no mask names hold NaN bytes; a row that sees a token beyond
    the format, a page that is not there or a slot past the table is NaN, and
    no other row is."""
    torch = torch_cuda()
    gen = np.random.default_rng(11)
    kv, group, r, pages = 2, 8, 20, 206  # 160 columns behind 13184 slots
    heads, n = kv * group, 206 * 64 - 2
    assert heads // kv * r * pages * 64 > MANY
    c = Cache(gen, dim, kv, 1, pages)
    k, v = _kv(gen, n, kv, dim)
    c.append(aa.F32, _dev(k[:n - 4]), _dev(v[:n - 4]), [0, n - 4], [n - 4])  # the last four are never written
    on = np.eye(r, dtype=bool)
    on[5, 2] = on[9, 7] = True
    on[16:] = False                                                     # and never seen
    q = _dev((3 * gen.standard_normal((r, heads * dim))).astype(np.float32), ty)
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
    want = np.zeros((r, heads), bool)
    want[[7, 9], group:] = True
    assert np.array_equal(torch.isnan(o2.view(r, heads, dim)).all(-1).cpu().numpy(), want)
    assert torch.equal(torch.isnan(l2).cpu(), torch.from_numpy(want))
    assert torch.equal(o2.view(r, heads, dim)[~torch.from_numpy(want)], out.view(r, heads, dim)[~torch.from_numpy(want)])
    # A page amid the cache is not there: rows whose window ends before it are as they were.
    t = c.host_table.copy()
    t[0, 100] = -1
    c.set_table(t)
    o3, _ = _tree_attend(c, ty, q, [0, r], [n], heads, 0.1, mask(on), 1)
    assert torch.isnan(o3).all()
    c.set_table(c.host_table)
    a, la = _tree_attend(c, ty, q, [0, r], [n], heads, 0.1, mask(on), 1, window=3000)
    c.set_table(t)
    b, lb = _tree_attend(c, ty, q, [0, r], [n], heads, 0.1, mask(on), 1, window=3000)
    assert torch.equal(torch.nan_to_num(a), torch.nan_to_num(b)) and torch.isnan(b).sum() == 2 * group * dim
    # Slots past the table.
    c.set_table(c.host_table)
    o5, _ = _tree_attend(c, ty, q, [0, r], [pages * 64 - 16 + r], heads, 0.1, mask(np.eye(r, dtype=bool)), 1)
    assert torch.isnan(o5[16:]).all()
    o7, _ = _tree_attend(c, ty, q, [0, r], [pages * 64 + 1 + r], heads, 0.1, mask(np.zeros((r, r), bool)), 1)
    assert torch.isnan(o7).all()


def test_captured_and_replayed():
    """One launch list for lengths and masks that change between replays, with other work in between."""
    torch = torch_cuda()
    gen = np.random.default_rng(3)
    rows, lens, heads = [40, 0, 25], [3000, 70, 5000], 16
    c = _widen(_filled(gen, 128, 2, [n + 200 for n in lens]), 320)
    starts = _starts(rows)
    q = _dev(gen.standard_normal((65, heads * 128)).astype(np.float32), aa.BF16)
    st, ln = _i32(starts), _i32(lens)
    mask = torch.zeros((65, 2), dtype=torch.int32, device="cuda")
    out, lse = torch.zeros_like(q), torch.zeros((65, heads), device="cuda")
    work = torch.empty(c.dev.kv4_tree_attention_work_bytes(c.c, heads, 65, 3, 40), dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()

    def run():
        c.dev.kv4_tree_attention(c.c, aa.BF16, q.data_ptr(), heads * 128, heads, 65, 3, st.data_ptr(), 40, ln.data_ptr(),
                                 mask.data_ptr(), 2, 0.1, out.data_ptr(), heads * 128, work.data_ptr(), stream(),
                                 lse=lse.data_ptr())

    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        run()
    for turn in range(4):
        now = [n + 50 * turn for n in lens]
        ons = [plain.ancestors(_forest(gen, r)) for r in rows]
        mask.copy_(_dev(np.concatenate([plain.mask_words(on, 2) if len(on) else np.zeros((0, 2), np.uint32) for on in ons]).view(np.int32)))
        ln.copy_(_i32(now))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        a, la = out.clone(), lse.clone()
        out.zero_()
        run()
        torch.cuda.synchronize()
        assert torch.equal(a, out) and torch.equal(la, lse)
        _check_tree(c, aa.BF16, q, starts, now, heads, 0.1, ons, 0, a, la)
