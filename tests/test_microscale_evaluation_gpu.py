"""A float weight without gradients: the training call's result, and none of
what it keeps for a backward pass."""
import pytest
import torch

from sym_b200 import microscale as mx
from sym_b200 import pyreloc

pytestmark = pytest.mark.gpu


def operands(m, n, k, dtype):
    g = torch.Generator().manual_seed(m)
    return (torch.randn(m, k, generator=g).to(dtype).cuda().requires_grad_(),
            torch.randn(n, k, generator=g).to(dtype).cuda().requires_grad_())


@pytest.mark.parametrize("dtype", (torch.float32, torch.float16, torch.bfloat16))
@pytest.mark.parametrize("m,n,k", [(1, 40, 100), (7, 300, 2048), (130, 257, 96), (700, 1030, 520)])
def test_result_is_the_training_calls(m, n, k, dtype):
    x, w = operands(m, n, k, dtype)
    want = mx.linear(x, w)
    assert want.requires_grad
    with torch.no_grad():
        y = mx.linear(x, w)
    assert not y.requires_grad and torch.equal(y, want)
    assert torch.equal(mx.linear(x.detach(), w.detach()), want)
    with torch.inference_mode():
        assert torch.equal(mx.linear(x, w, dtype=torch.float32), mx.linear(x.detach(), w.detach(), dtype=torch.float32))
    out = mx.linear(x.detach().view(1, m, k), w.detach().t().contiguous().t())
    assert torch.equal(out[0], want)


def test_nothing_is_kept_or_made_for_a_backward_pass():
    m, n, k = 2048, 4096, 4096
    x, w = operands(m, n, k, torch.bfloat16)
    mx.linear(x, w)
    torch.cuda.synchronize()

    def cost(call):
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before, launches = torch.cuda.memory_allocated(), pyreloc.kernel_launches()
        y = call()
        torch.cuda.synchronize()
        return torch.cuda.max_memory_allocated() - before, pyreloc.kernel_launches() - launches, y

    held = lambda r, c: r * c // 2 + r * c // 32  # noqa: E731  whole blocks and tiles here
    with torch.no_grad():
        peak, launches, _ = cost(lambda: mx.linear(x, w))
    assert launches == 3  # both operands quantised, their product
    assert peak <= 2 * m * n + held(m, k) + held(n, k) + 8 * 512 + (2 << 20)  # allocations are rounded up
    x1 = x.detach()[:1]
    with torch.no_grad():
        assert cost(lambda: mx.linear(x1, w))[1] <= 3


def test_no_rows_and_no_columns():
    with torch.no_grad():
        for m, n in ((0, 40), (5, 0), (0, 0)):
            x, w = operands(m, n, 64, torch.float16)
            assert mx.linear(x, w).shape == (m, n)
            assert mx.linear(x.view(1, m, 64), w).shape == (1, m, n)
