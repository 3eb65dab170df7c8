"""Sums so long that a tile takes more time than the wait limit, which is for a
step of it."""
import pytest
import torch

from sym_b200 import _native
from sym_b200 import microscale as mx

pytestmark = pytest.mark.gpu


def ones(rows, cols):
    return mx.MxTensor(torch.full((rows, cols // 2), 0x22, dtype=torch.uint8, device="cuda"),
                       torch.full((-(-rows // 128) * (cols // 128) * 512,), 127, dtype=torch.uint8, device="cuda"),
                       (rows, cols))


@pytest.mark.parametrize("m,n,k", [(1, 128, 1 << 25), (2048, 2048, 1 << 21)])
def test_the_limit_is_for_a_step(m, n, k):
    """Single CTAs (16,384 steps each) and pairs (8,192 steps a tile), both some
    milliseconds of work, under a limit of 0.2. The sum of k ones is exact."""
    a, b = ones(m, k), ones(n, k)
    limit = _native.cuda_layer().sbc_set_wait_limit_ns
    mx.check()
    limit(200_000)
    try:
        y = mx.matmul(a, b, dtype=torch.float32)
        mx.check()
    finally:
        limit(0)  # the default
    assert (y == k).all()
