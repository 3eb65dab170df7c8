"""Views whose values are not those of their memory: imaginary parts of
conjugated complex tensors are negated on reading."""
import pytest
import torch

from sym_b200 import microscale as mx

pytestmark = pytest.mark.gpu


def test_negated_views():
    g = torch.Generator().manual_seed(1)
    z = torch.randn(40, 64, dtype=torch.complex64, generator=g).cuda()
    w = torch.randn(96, 64, generator=g).cuda()
    q, qt = mx.quantize_both(w)
    column = torch.randn(40, 1, dtype=torch.complex64, generator=g).cuda()
    for v in (z.conj().imag, torch._neg_view(z.real.contiguous()), torch._neg_view(z.real.contiguous()).t(),
              column.conj().imag, torch._neg_view(z.real.contiguous())[0]):
        assert v.is_neg()
        plain = v.resolve_neg().clone()
        assert torch.equal(mx.quantize(v).codes, mx.quantize(plain).codes)
        if v.dim() == 2:
            assert torch.equal(mx.quantize(v, along=0).codes, mx.quantize(plain, along=0).codes)
            assert torch.equal(mx.quantize_both(v)[1].codes, mx.quantize_both(plain)[1].codes)
        assert torch.equal(mx.silu_mul(v, v), mx.silu_mul(plain, plain))
        if v.shape[-1] == 64:
            assert torch.equal(mx.linear(v, q), mx.linear(plain, q))
            assert torch.equal(mx.linear(v, torch._neg_view(w)), mx.linear(plain, -w))
    x = z.real.contiguous().requires_grad_()
    dy = torch.randn(40, 96, generator=g).cuda()
    for call in (lambda: mx.linear(x, q, qt), lambda: mx.linear(x, w)):
        got, = torch.autograd.grad(call(), x, torch._neg_view(dy))
        want, = torch.autograd.grad(call(), x, -dy)
        assert torch.equal(got, want)
    dh = torch.randn(40, 32, generator=g).cuda()
    got, = torch.autograd.grad(mx.silu_mul(x), x, torch._neg_view(dh))
    assert torch.equal(got, torch.autograd.grad(mx.silu_mul(x), x, -dh)[0])
