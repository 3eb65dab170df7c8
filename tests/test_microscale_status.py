"""A product whose bounded wait ran out is told to whom it concerns. The waits
run out by a withheld copy (10 ms) or are said to have by a host store."""
import ctypes

import pytest
import torch

from sym_b200 import _native, pyreloc
from sym_b200 import microscale as mx


def status(device):
    err = _native.SbError()
    rc = _native.lib().sb_mx_status(device, ctypes.byref(err))
    return rc, _native.error_of(err)[0] if rc else None


def test_status_without_products():
    assert status(0) == (0, None) and status(500) == (0, None)
    assert status(-1) == (1, "invalid_view")
    with pytest.raises(ValueError):
        mx.check("cpu")


def product(m=12):
    g = torch.Generator().manual_seed(m)
    x, w = torch.randn(m, 512, generator=g).cuda(), torch.randn(300, 512, generator=g).cuda()
    return x, mx.quantize(w)


@pytest.mark.gpu
@pytest.mark.parametrize("m", (1, 12, 300))
def test_last_product_is_reported_on_request(m):
    x, q = product(m)
    want = mx.linear(x, q)
    mx.check()
    _native.cuda_layer().sbc_test_withhold_mx(10_000_000)
    mx.linear(x, q)
    with pytest.raises(pyreloc.TransferError) as e:
        mx.check(x.device)
    assert e.value.code == "backend_failure"
    for device in (None, 0, "cuda", "cuda:0"):
        mx.check(device)  # reported once
    assert torch.equal(mx.linear(x, q), want)


@pytest.mark.gpu
def test_replays_are_reported_on_request():
    x, q = product()
    want = mx.linear(x, q)
    torch.cuda.synchronize()
    graphs = []
    for withhold in (0, 10_000_000):
        _native.cuda_layer().sbc_test_withhold_mx(withhold)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = mx.linear(x, q)
        graphs.append((g, y))
    for _ in range(2):
        graphs[0][0].replay()
        mx.check()
        assert torch.equal(graphs[0][1], want)
        graphs[1][0].replay()
        with pytest.raises(pyreloc.TransferError):
            mx.check()


@pytest.mark.gpu
def test_a_fault_concerns_its_own_device():
    x, q = product()
    want = mx.linear(x, q)
    mx.check()
    hooks = _native.cuda_layer()
    hooks.sbc_test_mx_fault(1)
    assert torch.equal(mx.linear(x, q), want)
    mx.check(0)
    assert status(1) == (1, "backend_failure") and status(1) == (0, None)
    hooks.sbc_test_mx_fault(0)
    assert status(1) == (0, None)
    with pytest.raises(pyreloc.TransferError):
        mx.matmul(q, q)
    hooks.sbc_test_mx_fault(63)
    hooks.sbc_test_mx_fault(200)  # devices from 63 on share a word
    assert status(64) == (1, "backend_failure") and status(63) == (0, None)
    mx.check()
