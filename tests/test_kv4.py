"""CPU checks of the rotary and 4-bit cache calls: rotation tables, sizes,
and refusals, which come before any GPU work."""
import ctypes
import errno

import numpy as np
import pytest

import aspida_amd as aa
import kv4_plain as plain

P16 = 1 << 20  # addresses that are never followed


@pytest.fixture(scope="module")
def lib():
    return aa.load()


@pytest.mark.parametrize("kw", [
    dict(rot_dim=128, base=500000.0),
    dict(rot_dim=2, base=10000.0),
    dict(rot_dim=256, base=10000.0, scaling="linear", factor=4.0),
    dict(rot_dim=128, base=500000.0, scaling="bands", factor=8.0, low=1.0, high=4.0, context=8192),
    dict(rot_dim=64, base=1000000.0, scaling="yarn", factor=4.0, low=1.0, high=32.0, context=32768),
    dict(rot_dim=96, base=10000.0, scaling="yarn", factor=16.0, low=1.0, high=32.0, context=4096),
    dict(rot_dim=8, base=10000.0, freq_factors=[1.0, 1.5, 4.0, 8.0]),
    dict(rot_dim=8, base=10000.0, scaling="linear", factor=2.0, freq_factors=[1.0, 1.5, 4.0, 8.0]),
], ids=str)
def test_rotation_table(kw, lib):
    r = aa.Rope(**kw)
    f, mag = r.table()
    args = dict(kw)
    want = plain.rope_freqs(args.pop("rot_dim"), args.pop("base"), **args)
    # A handful of f64 operations and pow, each to about an ulp.
    assert np.all(np.abs(f - want) <= 16 * 2.0 ** -53 * want)
    if kw.get("scaling") == "yarn":
        assert abs(mag - (0.1 * np.log(kw["factor"]) + 1)) < 1e-15
    else:
        assert mag == 1.0
    assert aa.Rope(64, magnitude=0.75, scaling="yarn", factor=4.0, high=32.0, context=4096).table()[1] == 0.75
    r.close()
    r.close()


@pytest.mark.parametrize("kw", [
    dict(rot_dim=0), dict(rot_dim=3), dict(rot_dim=258), dict(rot_dim=-2), dict(rot_dim=64, base=1.0),
    dict(rot_dim=64, base=float("nan")), dict(rot_dim=64, base=float("inf")),
    dict(rot_dim=64, scaling="linear", factor=0.0), dict(rot_dim=64, scaling="linear", factor=float("nan")),
    dict(rot_dim=64, scaling="bands", factor=2.0, low=4.0, high=4.0, context=10),
    dict(rot_dim=64, scaling="yarn", factor=2.0, low=0.0, high=4.0, context=10),
    dict(rot_dim=64, scaling="yarn", factor=2.0, context=0), dict(rot_dim=64, magnitude=-1.0),
    dict(rot_dim=64, magnitude=float("inf")), dict(rot_dim=4, freq_factors=[1.0, 0.0]),
    dict(rot_dim=4, freq_factors=[1.0, float("nan")]),
], ids=str)
def test_bad_rotations_are_refused(kw, lib):
    with pytest.raises(RuntimeError):
        aa.Rope(**kw)
    assert lib.aspida_gpu_last_error() == 0  # the constructor took it


def test_rope_constructor_checks_names(lib):
    for kw in (dict(layout="rows"), dict(scaling="cubic"), dict(freq_factors=[1.0])):
        with pytest.raises(ValueError):
            aa.Rope(64, **kw)
    assert lib.aspida_rope_create(None) is None and lib.aspida_gpu_last_error() != 0
    bad = aa._RopeParams(64, 0, 4, 0, 1e4, 1, 1, 1, 1, 0, None)
    assert lib.aspida_rope_create(ctypes.byref(bad)) is None and lib.aspida_gpu_last_error() != 0


def test_page_bytes(lib):
    for d in (64, 128, 256):
        assert lib.aspida_kv4_page_bytes(d, 8) == 80 * d * 8
    for d, n in ((0, 1), (96, 1), (80, 1), (512, 1), (128, 0), (128, 65536)):
        assert lib.aspida_kv4_page_bytes(d, n) == 0


def _rope_call(lib, **kw):
    r = kw.pop("rope", None) or aa.Rope(kw.pop("rot", 64))
    a = dict(type=0, x=P16, xs=256, n=1, heads=2, dim=128, pos=P16, inv=0, y=2 * P16, ys=256)
    a.update(kw)
    return lib.aspida_rope_dev(r.h, *a.values(), None)


@pytest.mark.parametrize("kw", [
    dict(type=3), dict(type=-1), dict(x=None), dict(x=P16 + 2), dict(xs=255), dict(n=-1), dict(heads=0),
    dict(heads=65536, xs=1 << 30, ys=1 << 30), dict(dim=32), dict(pos=None), dict(pos=P16 + 1), dict(y=None),
    dict(ys=255), dict(y=P16, ys=512), dict(type=1, x=P16 + 1),
], ids=str)
def test_rope_refusals(kw, lib):
    assert _rope_call(lib, **kw) == -errno.EINVAL


def test_rope_without_tokens_and_without_a_form(lib):
    assert _rope_call(lib, n=0) == 0
    assert lib.aspida_rope_dev(None, 0, P16, 256, 1, 2, 128, P16, 0, P16, 256, None) == -errno.EINVAL
    # 1000 + 31 single values: more than 256 pieces of any width that divides both.
    assert _rope_call(lib, rot=62, dim=1062, heads=1, xs=2000, ys=2000) == -errno.ENOTSUP


def _cache(**kw):
    a = dict(head_dim=128, n_kv=2, n_pages=4, max_pages=3, pages=P16, table=P16)
    a.update(kw)
    return aa.KV4Cache(*a.values())


BAD_CACHES = [dict(head_dim=96), dict(head_dim=0), dict(n_kv=0), dict(n_kv=65536), dict(n_pages=0), dict(max_pages=0),
              dict(max_pages=(1 << 24) + 1), dict(pages=None), dict(pages=P16 + 8), dict(table=None),
              dict(table=P16 + 2)]
ROWS = dict(n_rows=2, n_seq=2, row_start=None, kv_len=P16)
BAD_ROWS = [dict(n_rows=-1), dict(n_seq=-1), dict(n_seq=65536, n_rows=65536), dict(kv_len=None), dict(kv_len=P16 + 1),
            dict(n_rows=3), dict(row_start=P16 + 2)]


def _append(lib, cache=None, rope=None, pos=None, **kw):
    a = dict(type=0, k=P16, ks=256, v=P16, vs=256, **ROWS)
    a.update(kw)
    return lib.aspida_kv4_append_dev((cache or _cache()).ref, *a.values(), rope, pos, None)


def _read(lib, cache=None, **kw):
    a = dict(type=0, **ROWS, k=P16, ks=256, v=P16, vs=256)
    a.update(kw)
    return lib.aspida_kv4_read_dev((cache or _cache()).ref, *a.values(), None)


def _attn(lib, cache=None, **kw):
    a = dict(type=0, q=P16, qs=1024, heads=8, n_rows=2, n_seq=2, row_start=None, max_rows=1, kv_len=P16, scale=0.1,
             window=0, out=P16, os=1024, lse=None, work=P16)
    a.update(kw)
    return lib.aspida_kv4_attn_dev((cache or _cache()).ref, *a.values(), None)


def _weigh(lib, cache=None, **kw):
    a = dict(type=0, q=P16, qs=1024, heads=8, n_rows=2, n_seq=2, row_start=None, max_rows=1, kv_len=P16, scale=0.1,
             window=0, lse=P16, acc_in=None, acc_out=P16, stride=64)
    a.update(kw)
    return lib.aspida_kv4_weigh_dev((cache or _cache()).ref, *a.values(), None)


@pytest.mark.parametrize("call", [_append, _read, _attn, _weigh], ids=lambda f: f.__name__)
def test_cache_calls_refuse_bad_caches_rows_and_types(call, lib):
    for kw in BAD_CACHES:
        assert call(lib, cache=_cache(**kw)) == -errno.EINVAL, kw
    for kw in BAD_ROWS + [dict(type=3), dict(type=-1)]:
        assert call(lib, **kw) == -errno.EINVAL, kw
    assert call(lib, n_rows=0) == 0 and call(lib, n_rows=0, n_seq=0) == 0
    assert lib.aspida_gpu_last_error() == 0


def test_append_and_read_refusals(lib):
    for kw in (dict(k=None), dict(v=None), dict(ks=255), dict(vs=255), dict(k=P16 + 2), dict(type=2, v=P16 + 1)):
        assert _append(lib, **kw) == -errno.EINVAL, kw
        assert _read(lib, **kw) == -errno.EINVAL, kw
    assert _append(lib, rope=aa.Rope(64).h, pos=None) == -errno.EINVAL
    assert _append(lib, rope=aa.Rope(130).h, pos=P16) == -errno.EINVAL


def test_attention_and_weigh_refusals(lib):
    both = [dict(q=None), dict(q=P16 + 2), dict(qs=1023), dict(heads=0), dict(heads=7), dict(max_rows=0),
            dict(scale=float("nan")), dict(scale=float("inf")), dict(window=-1)]
    for kw in both + [dict(out=None), dict(os=1023), dict(lse=P16 + 2), dict(work=None), dict(work=P16 + 128)]:
        assert _attn(lib, **kw) == -errno.EINVAL, kw
    for kw in both + [dict(lse=None), dict(acc_in=P16 + 2), dict(acc_out=None), dict(stride=0)]:
        assert _weigh(lib, **kw) == -errno.EINVAL, kw
    dev, c = aa.DeviceOps(), _cache()
    assert dev.kv4_attention_work_bytes(c, 8, 2, 2, 1) > 0
    for args in ((7, 2, 2, 1), (8, -1, 2, 1), (8, 2, -1, 1), (8, 2, 2, 0)):
        with pytest.raises(ValueError):
            dev.kv4_attention_work_bytes(c, *args)
    with pytest.raises(RuntimeError):
        dev.kv4_attention(c, 0, 0, 1024, 8, 2, 2, 0, 1, P16, 0.1, P16, 1024, P16)


def test_evict_refusals(lib):
    def call(src=None, dst=None, **kw):
        a = dict(n_seq=2, kv_len=P16, acc=P16, stride=192, keep=128, first=4, recent=16)
        b = dict(new_len=P16, idx=P16, acc_out=P16)
        a.update({k: v for k, v in kw.items() if k in a})
        b.update({k: v for k, v in kw.items() if k in b})
        return lib.aspida_kv4_evict_dev((src or _cache()).ref, *a.values(), (dst or _cache(pages=2 * P16)).ref,
                                        *b.values(), None)
    for kw in (dict(n_seq=-1), dict(n_seq=65536), dict(kv_len=None), dict(acc=None), dict(stride=0), dict(keep=0),
               dict(first=-1), dict(recent=-1), dict(first=100, recent=29), dict(keep=193), dict(new_len=None),
               dict(idx=None), dict(acc_out=P16 + 1)):
        assert call(**kw) == -errno.EINVAL, kw
    for kw in BAD_CACHES:
        assert call(src=_cache(**kw)) == -errno.EINVAL and call(dst=_cache(**kw)) == -errno.EINVAL, kw
    assert call(dst=_cache(n_kv=1)) == -errno.EINVAL and call(dst=_cache(head_dim=64)) == -errno.EINVAL
    assert call(n_seq=0) == 0


def test_plain_quantiser_on_known_values():
    """The step is the range / 15 rounded up to 7 bits; ties go to even codes."""
    x = np.zeros(32, np.float32)
    x[:3] = [0, 15, 0.5]
    d, m, q = plain.quantise(x)
    assert d == 1 and m == 0 and list(q[0][:3]) == [0, 15, 0]
    x[1] = 15.01
    d, _, _ = plain.quantise(x)
    assert d == 1 + 2.0 ** -6
    assert np.all(plain.stands_for(np.full(32, 3.0, np.float32)) == 3.0)
    x[4] = np.inf
    assert np.isnan(plain.stands_for(x)).all()
