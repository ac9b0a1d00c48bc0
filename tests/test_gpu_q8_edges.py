"""The 8-bit KV cache at the ends of what its definition allows."""
import numpy as np
import pytest
import torch

from tests import q_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def nn():
    from tests.helpers import build_library
    build_library()
    from alpakann_b200.onHost import nn
    return nn


@pytest.mark.parametrize("D", [64, 5])
@pytest.mark.parametrize("grow", [1e-3, 50.0])
def test_append_behind_a_negative_scale(nn, D, grow):
    """Rows appended into a block whose scale is negative: what the earlier tokens stand
    for stays, exactly where the scale's size does, else to half a step of the new one."""
    g = np.random.default_rng(D)
    kc, ks = ref.make_cache(g, 2, 2, 40, D, 16)
    ks *= np.array([1, -1, -1], np.float32)
    dev = [torch.from_numpy(a).cuda() for a in (kc, kc, ks, ks)]
    x = torch.from_numpy((g.standard_normal((2, 3, 2, D)) * grow).astype(np.float32)).cuda()
    before, after = (torch.zeros(2, 2, 2, 40, D, device="cuda") for _ in range(2))
    nn.kvCacheReadQ8(None, None, *dev, before[0], before[1], 16)
    starts = [20, 33]
    nn.kvCacheAppendQ8(None, None, x, x, *dev, torch.tensor(starts, dtype=torch.int32, device="cuda"), 16)
    nn.kvCacheReadQ8(None, None, *dev, after[0], after[1], 16)
    for b, n in enumerate(starts):
        scale = dev[2][b, :, n // 16, None, None]
        assert (scale > 0).all()
        old, new = before[0, b, :, :n], after[0, b, :, :n]
        if grow < 1:
            assert torch.equal(old, new)
        else:  # half a step, and the 64-bit quotient's and the read-back's roundings
            assert ((old - new).abs() <= 0.5001 * scale)[:, n // 16 * 16:].all()
            assert torch.equal(old[:, :n // 16 * 16], new[:, :n // 16 * 16])
        assert ((after[0, b, :, n:n + 3] - x[b].transpose(0, 1)).abs() <= 0.5001 * scale).all()
    assert torch.equal(after[0], after[1])


def test_append_into_a_cache_of_no_tokens_is_reported(nn):
    import alpakann_b200 as ann
    from alpakann_b200 import _capi
    queue = ann.Queue()
    queue.take_device_error()
    cache, scale = torch.zeros(2, 3, 0, 64, dtype=torch.int8, device="cuda"), torch.zeros(2, 3, 0, device="cuda")
    x, pos = torch.randn(2, 4, 3, 64, device="cuda"), torch.tensor([0, 5], dtype=torch.int32, device="cuda")
    args = (x, x, cache, cache, scale, scale, pos, 16)
    nn.kvCacheAppendQ8(None, None, *args, counts=torch.zeros(2, dtype=torch.int32, device="cuda"))
    assert queue.take_device_error() == 0  # no rows, none dropped
    nn.kvCacheAppendQ8(None, None, *args)
    assert queue.take_device_error() == _capi.ANN_DEVERR_CACHE_RANGE
