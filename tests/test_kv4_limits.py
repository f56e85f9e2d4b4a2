"""CPU checks of the 4-bit cache calls at the edges of what they allow."""
import pytest

import aspida_amd as aa

P16 = 1 << 20  # an address that is never followed


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_one_attention_workspace_serves_every_call(dim):
    """Two parts of 16 columns of 4 dim + 8 bytes for each workgroup that the
    card holds at once, whatever the rows and sequences."""
    dev, c = aa.DeviceOps(), aa.KV4Cache(dim, 8, 4, 3, P16, P16)
    want = 2 * {64: 768, 128: 512, 256: 256}[dim] * 16 * (4 * dim + 8)
    for args in ((32, 1, 1, 1), (64, 64, 64, 1), (64, 9000, 3, 4097), (64, 9000, 3, 2 ** 31 - 1), (32, 32768, 1, 32768),
                 (64, 65536, 16, 4096), (64, 4159, 64, 4096), (64, 263, 64, 200), (65528, 2 ** 31 - 1, 65535, 2 ** 31 - 1)):
        assert dev.kv4_attention_work_bytes(c, *args) == want


def test_a_closed_rotation_is_refused():
    """Also where no rotation is a choice: keys are not stored unrotated by mistake."""
    dev, c, rope = aa.DeviceOps(), aa.KV4Cache(128, 2, 4, 3, P16, P16), aa.Rope(64)
    rope.close()
    with pytest.raises(ValueError):
        rope.table()
    with pytest.raises(ValueError):
        dev.rope(rope, aa.F32, P16, 256, 0, 2, 128, P16, P16, 256)
    with pytest.raises(ValueError):
        dev.kv4_append(c, aa.F32, P16, 256, P16, 256, 0, 0, 0, P16, rope, P16)  # no rows: nothing is followed


@pytest.mark.parametrize("kw", [dict(freq_factors=[1e-30, 1.0]), dict(freq_factors=[1.0, 1e-12]),
                                dict(scaling="linear", factor=2.0 ** -19 * 0.999), dict(scaling="linear", factor=1e-300),
                                dict(scaling="yarn", factor=1e-9, low=1.0, high=32.0, context=4096)], ids=str)
def test_rotations_too_fast_for_their_angles_are_refused(kw):
    with pytest.raises(RuntimeError):
        aa.Rope(4, **kw)
    assert aa.load().aspida_gpu_last_error() == 0  # the constructor took it


def test_the_fastest_rotation():
    assert aa.Rope(4, scaling="linear", factor=2.0 ** -19).table()[0][0] == 2.0 ** 19
