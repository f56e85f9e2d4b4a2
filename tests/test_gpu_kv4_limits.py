"""The 4-bit cache calls at the edges of what their contracts allow."""
import numpy as np
import pytest

from gpu_helpers import stream, sync, torch_cuda
from test_gpu_kv4 import Cache, _dev, _filled, _i32

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
