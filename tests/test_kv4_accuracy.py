"""The limits of kv4_accuracy.py: kept by two f16 numbers for each query value
and softmax weight, broken by one.  CPU only: the oracle's own arithmetic."""
import numpy as np
import pytest

import kv4_accuracy as acc
import kv4_plain as plain

# dim, heads, kv, rows, slots, window: as test_gpu_kv4_accuracy.py has them
SHAPES = [(128, 32, 8, 1, 3000, 0), (64, 8, 2, 3, 700, 0), (256, 8, 4, 2, 500, 100), (128, 8, 2, 100, 400, 0)]


def _case(shape):
    dim, heads, kv, rows, n, window = shape
    gen = np.random.default_rng(dim + rows)
    k = gen.standard_normal((n, kv, dim)) * np.exp(0.7 * gen.standard_normal((kv, dim))) + gen.standard_normal((kv, dim))
    k, v = plain.stands_for(k.astype(np.float32)), plain.stands_for(gen.standard_normal((n, kv, dim)).astype(np.float32))
    q = (2 * gen.standard_normal((rows, heads, dim))).astype(np.float32).astype(np.float64)
    return q, k, v, dim ** -0.5, window


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_f32_limits_tell_one_plane_from_two(shape):
    q, k, v, scale, window = _case(shape)
    want, wl, _, _ = plain.attend(q, k, v, scale, window)
    o32, l32 = acc.attend32(q, k, v, scale, window)
    out, lse = acc.attend_planes(q, k, v, scale, 2, 2, window)
    assert acc.over(out, want, o32) < 1 and acc.over(lse, wl, l32) < 1
    assert acc.over(acc.attend_planes(q, k, v, scale, 2, 1, window)[0], want, o32) > 1
    out, lse = acc.attend_planes(q, k, v, scale, 1, 2, window)
    assert acc.over(out, want, o32) > 1 and acc.over(lse, wl, l32) > 1


@pytest.mark.parametrize("bits", [8, 11], ids=["bf16", "f16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_16_bit_limits_tell_one_plane_from_two(shape, bits):
    q, k, v, scale, window = _case(shape)
    q = acc.round16(q, bits)[0]
    want = plain.attend(q, k, v, scale, window)[0]
    o32 = acc.attend32(q, k, v, scale, window)[0]
    two = acc.round16(acc.attend_planes(q, k, v, scale, 2, 2, window)[0], bits)[0]
    one = acc.round16(acc.attend_planes(q, k, v, scale, 2, 1, window)[0], bits)[0]
    assert acc.over16(two, want, o32, bits) < 1 < acc.over16(one, want, o32, bits)


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_slot_weight_limits_tell_one_plane_from_two(shape):
    q, k, v, scale, window = _case(shape)
    lse = plain.attend(q, k, v, scale, window)[1].astype(np.float32).astype(np.float64)
    want, w32 = plain.weights(q, k, lse, scale, window), acc.weights32(q, k, lse, scale, window)
    some = want > 0
    for n, good in ((2, True), (1, False)):
        got = plain.weights(acc.query_planes(q, n), k, lse, scale, window)
        assert (acc.over(got[some] / want[some], 1.0, w32[some] / want[some]) < 1) == good
