"""CPU checks of the tree calls and the 8-bit integer products: sizes,
refusals (which come before any GPU work), and the plain forms."""
import errno

import numpy as np
import pytest

import aspida_amd as aa
import more_plain as plain
from test_kv4 import BAD_CACHES, BAD_ROWS, P16, ROWS, _cache


@pytest.fixture(scope="module")
def lib():
    return aa.load()


def _tree(lib, **kw):
    a = dict(parent=P16, **ROWS, pos=P16, mask=P16, words=1)
    a.update(kw)
    return lib.aspida_tree_dev(*a.values(), None)


def _accept(lib, **kw):
    a = dict(type=0, logits=P16, stride=100, vocab=100, **ROWS, parent=P16, token=P16, path=P16, count=P16, next=P16,
             new_len=P16, work=P16)
    a.update(kw)
    return lib.aspida_tree_accept_dev(*a.values(), None)


def _keep(lib, cache=None, **kw):
    a = dict(**ROWS, path=P16, count=P16)
    a.update(kw)
    return lib.aspida_kv4_keep_dev((cache or _cache()).ref, *a.values(), None)


def _attn(lib, cache=None, **kw):
    a = dict(type=0, q=P16, qs=1024, heads=8, n_rows=2, n_seq=2, row_start=None, max_rows=1, kv_len=P16, mask=P16,
             words=1, scale=0.1, window=0, out=P16, os=1024, lse=None, work=P16)
    a.update(kw)
    return lib.aspida_kv4_tree_attn_dev((cache or _cache()).ref, *a.values(), None)


@pytest.mark.parametrize("call", [_tree, _accept, _keep, _attn], ids=lambda f: f.__name__)
def test_tree_calls_refuse_bad_rows(call, lib):
    for kw in BAD_ROWS:
        assert call(lib, **kw) == -errno.EINVAL, kw
    assert call(lib, n_rows=0) == 0 and call(lib, n_rows=0, n_seq=0) == 0
    assert lib.aspida_gpu_last_error() == 0


@pytest.mark.parametrize("call", [_keep, _attn], ids=lambda f: f.__name__)
def test_tree_calls_refuse_bad_caches(call, lib):
    for kw in BAD_CACHES:
        assert call(lib, cache=_cache(**kw)) == -errno.EINVAL, kw


def test_tree_refusals(lib):
    for kw in (dict(parent=None), dict(parent=P16 + 2), dict(pos=P16 + 1), dict(mask=P16 + 2), dict(words=0),
               dict(words=129)):
        assert _tree(lib, **kw) == -errno.EINVAL, kw
    for kw in (dict(path=None), dict(path=P16 + 2), dict(count=None), dict(count=P16 + 1)):
        assert _keep(lib, **kw) == -errno.EINVAL, kw


def test_tree_attention_refusals(lib):
    for kw in (dict(q=None), dict(q=P16 + 2), dict(qs=1023), dict(heads=0), dict(heads=7), dict(max_rows=0),
               dict(max_rows=4097), dict(scale=float("nan")), dict(scale=float("inf")), dict(window=-1), dict(out=None),
               dict(os=1023), dict(lse=P16 + 2), dict(work=None), dict(work=P16 + 128), dict(mask=None),
               dict(mask=P16 + 2), dict(words=0), dict(words=129), dict(type=3), dict(type=-1)):
        assert _attn(lib, **kw) == -errno.EINVAL, kw
    dev, c = aa.DeviceOps(), _cache()
    assert dev.kv4_tree_attention_work_bytes(c, 8, 2, 2, 1) > 0
    for args in ((7, 2, 2, 1), (8, -1, 2, 1), (8, 2, -1, 1), (8, 2, 2, 0), (8, 2, 2, 4097)):
        with pytest.raises(ValueError):
            dev.kv4_tree_attention_work_bytes(c, *args)
    with pytest.raises(RuntimeError):
        dev.kv4_tree_attention(c, 0, 0, 1024, 8, 2, 2, 0, 1, P16, P16, 1, 0.1, P16, 1024, P16)


def test_accept_refusals(lib):
    for kw in (dict(type=3), dict(type=-1), dict(logits=None), dict(logits=P16 + 2), dict(stride=99), dict(vocab=0),
               dict(vocab=(1 << 30) + 1, stride=1 << 31), dict(parent=None), dict(token=None), dict(token=P16 + 2),
               dict(path=None), dict(count=None), dict(next=None), dict(new_len=None), dict(new_len=P16 + 2),
               dict(work=None), dict(work=P16 + 4), dict(n_rows=(1 << 22) + 1, row_start=P16)):
        assert _accept(lib, **kw) == -errno.EINVAL, kw
    dev = aa.DeviceOps()
    assert dev.tree_accept_work_bytes(0, 5) > 0
    for args in ((-1, 10), (1, 0), ((1 << 22) + 1, 10), (1, (1 << 30) + 1)):
        with pytest.raises(ValueError):
            dev.tree_accept_work_bytes(*args)


def _matmul(lib, **kw):
    a = dict(w=P16, in_dim=100, out_dim=10, type=0, x=P16, xs=100, n=2, y=2 * P16, ys=10, work=P16)
    a.update(kw)
    return lib.aspida_w8_matmul_dev(*a.values(), None)


def _gated(lib, **kw):
    a = dict(w=P16, up=P16, in_dim=100, out_dim=10, act=0, type=0, x=P16, xs=100, n=2, y=2 * P16, ys=10, work=P16)
    a.update(kw)
    return lib.aspida_w8_gated_dev(*a.values(), None)


@pytest.mark.parametrize("call", [_matmul, _gated], ids=lambda f: f.__name__)
def test_product_refusals(call, lib):
    for kw in (dict(w=None), dict(w=P16 + 8), dict(in_dim=0), dict(in_dim=131073, xs=131073), dict(out_dim=0),
               dict(out_dim=(1 << 22) + 1, ys=1 << 23), dict(type=3), dict(type=-1), dict(x=None), dict(x=P16 + 2),
               dict(xs=99), dict(n=-1), dict(n=(1 << 22) + 1), dict(y=None), dict(y=P16), dict(ys=9), dict(work=None),
               dict(work=P16 + 128), dict(type=1, x=P16 + 1), dict(n=1 << 20, out_dim=1 << 20, ys=1 << 20)):
        assert call(lib, **kw) == -errno.EINVAL, kw
    assert call(lib, n=0) == 0 and lib.aspida_gpu_last_error() == 0


def test_gated_and_packing_refusals(lib):
    for kw in (dict(up=None), dict(up=P16 + 8), dict(act=-1), dict(act=2)):
        assert _gated(lib, **kw) == -errno.EINVAL, kw
    pack = lambda **kw: lib.aspida_w8_pack_dev(*{**dict(c=P16, st=100, s=P16, i=100, o=10, p=P16), **kw}.values(), None)  # noqa: E731
    for kw in (dict(c=None), dict(st=99), dict(s=None), dict(s=P16 + 2), dict(i=0), dict(o=0), dict(p=None), dict(p=P16 + 8)):
        assert pack(**kw) == -errno.EINVAL, kw
    conv = lambda **kw: lib.aspida_w8_convert_dev(*{**dict(k=0, w=P16, i=256, o=10, p=P16), **kw}.values(), None)  # noqa: E731
    for kw in (dict(k=-2), dict(k=6), dict(i=100), dict(i=0), dict(o=0), dict(w=None), dict(k=-1, w=P16 + 2), dict(p=None)):
        assert conv(**kw) == -errno.EINVAL, kw
    assert lib.aspida_w8_unpack_dev(P16, 0, 1, P16, None) == -errno.EINVAL
    assert lib.aspida_w8_unpack_dev(P16, 1, 1, None, None) == -errno.EINVAL
    dev = aa.DeviceOps()
    assert dev.w8_bytes(1, 1) > 0 and dev.w8_work_bytes(0, 1) > 0
    assert dev.w8_bytes(4096, 4096) >= 4096 * (4096 + 4)
    for f, args in ((dev.w8_bytes, (0, 1)), (dev.w8_bytes, (131073, 1)), (dev.w8_bytes, (1, 0)),
                    (dev.w8_work_bytes, (-1, 1)), (dev.w8_work_bytes, (1, 0))):
        with pytest.raises(ValueError):
            f(*args)


def test_plain_forms_on_known_values():
    on = plain.ancestors([-1, 0, 0, 2, 7, 1])
    assert [list(np.nonzero(r)[0]) for r in on] == [[0], [0, 1], [0, 2], [0, 2, 3], [4], [0, 1, 5]]
    assert list(plain.mask_words(on, 1)[:, 0]) == [1, 3, 5, 13, 16, 35]
    see = plain.tree_sees(on, 3, 0)
    assert list(np.nonzero(see[3])[0]) == [0, 1, 2, 3, 5, 6]
    assert list(np.nonzero(plain.tree_sees(on, 3, 4)[3])[0]) == [2, 3, 5, 6]
    assert list(np.nonzero(plain.tree_sees(on, 3, 2)[3])[0]) == [3, 5, 6]
    assert list(np.nonzero(plain.tree_sees(on, -1, 0)[3])[0]) == [1, 2]
    logits = np.zeros((4, 5))
    logits[0, 3], logits[1, 1], logits[3, [2, 4]] = 1, np.nan, 7
    assert plain.accept(logits, [-1, 0, 0, 2], [0, 9, 3, 0]) == ([0, 2, 3], 2)
    s, c = plain.quantise8(np.float32([[127, 0.5, 1.5, -2.5, 126.5], [0, 0, 0, 0, 1e-31], [1, np.inf, 0, 0, 0]]))
    assert list(c[0]) == [127, 0, 2, -2, 126] and s[0] == 1 and s[1] == 0 and np.isnan(s[2])
