"""Every kernel variant that a microscaled product may take: the shapes below
reach each of them (checked without a GPU, on the SM count of a B200), and are
compared with the definition on the GPU.

Tolerance: that of test_microscale_gpu.check_product (terms exact in 32 bits, K
additions of at most a unit in the last place each, one rounding to the result)."""
import ctypes

import mx_oracle as O
import numpy as np
import pytest
import torch
from test_microscale_gpu import HALF_STEP, host, tensor

from sym_b200 import _native, pyreloc
from sym_b200 import microscale as mx

SMS = 148
# pairs of SMs: tiles of 256, 192 and 128 rows, one tile a pair up to seven
# (so that each of two accumulators is used again and again); then single CTAs
PAIRS = [(1003, 4101, 520), (1347, 9703, 66), (2737, 8767, 65), (300, 9001, 520), (777, 11008, 512),
         (1110, 11371, 67), (1468, 9525, 1000), (1822, 11893, 67), (163, 768, 68), (831, 7618, 520),
         (1541, 8364, 520)]
SINGLES = [(1, 512, 2048), (3, 700, 500), (8, 2000, 4096), (2, 5000, 200), (7, 19500, 500), (13, 20000, 100),
           (16, 900, 4096), (32, 300, 1000), (30, 19000, 64), (64, 1000, 4096), (50, 19001, 96), (128, 384, 768),
           (100, 18944, 130), (180, 300, 4000), (523, 7936, 164)]


def choice(m, n, k, sms=SMS):
    c = _native.SbcMxChoice()
    assert _native.cuda_layer().sbc_test_mx_plan(m, n, k, sms, ctypes.byref(c)) == 0
    return c


def test_the_shapes_reach_every_variant():
    pairs = [choice(*s) for s in PAIRS]
    for width in (256, 192, 128):
        turns = {c.turns for c in pairs if c.pair == width}
        assert 1 in turns and max(turns) >= 4 and len(turns) >= 3, (width, turns)
    singles = [choice(*s) for s in SINGLES]
    assert all(c.pair == 0 for c in singles)
    assert {(c.single, c.split > 1) for c in singles if not c.fused} == {
        (width, split) for width in (8, 16, 32, 64, 128) for split in (False, True)}
    assert {c.split > 1 for c in singles if c.fused} == {False, True}
    assert any(c.split == 8 for c in singles)


def test_sizes_past_the_copies_coordinates_are_refused():
    c = _native.SbcMxChoice()
    plan = _native.cuda_layer().sbc_test_mx_plan
    for m, n, k in ((2 ** 31 - 1, 128, 64), (1, 2 ** 31 - 1, 64), (1, 128, 2 ** 31), (2 ** 30, 2 ** 30, 64),
                    (0, 1, 1), (1, 0, 1), (1, 1, 0)):
        assert plan(m, n, k, SMS, ctypes.byref(c)) != 0
    assert plan(1, 1, 1, SMS, None) != 0 and plan(1, 1, 1, 0, ctypes.byref(c)) != 0


def operands(m, n, k):
    return tensor((m, k), torch.bfloat16, 80), tensor((n, k), torch.float32, 81, 0.02)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", PAIRS + SINGLES)
def test_products_of_every_variant(m, n, k):
    x, w = operands(m, n, k)
    q = mx.quantize(w)
    a, b = (torch.from_numpy(O.rounded(host(v))).cuda() for v in (x, w))
    want, size = a @ b.t(), a.abs() @ b.abs().t()
    for t in (torch.bfloat16, torch.float16, torch.float32):
        y = mx.linear(x, q, dtype=t)
        half = HALF_STEP[t]
        floor = torch.finfo(t).smallest_normal * half
        off = (y.double() - want).abs() - (k * 2.0 ** -23 * size * (1 + half) + half * want.abs() + floor)
        assert off.max().item() <= 0, off.max().item()
        assert torch.equal(y, mx.linear(x, q, dtype=t))
        assert torch.equal(y, mx.matmul(mx.quantize(x), q, dtype=t))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", (torch.float16, torch.float32))
@pytest.mark.parametrize("m,n,k", PAIRS[1:2] + PAIRS[4:5] + PAIRS[9:] + SINGLES)
def test_waits_that_run_out_end_every_variant(m, n, k, dtype):
    """The first copy of codes withheld: the kernel's bounded waits run out in
    the loading, multiplying and storing warps, it leaves by itself, the next
    product reports it and the one after is right."""
    x, w = operands(m, n, k)
    q = mx.quantize(w)
    want = mx.linear(x, q, dtype=dtype)
    torch.cuda.synchronize()
    _native.cuda_layer().sbc_test_withhold_mx(10_000_000)
    mx.linear(x, q, dtype=dtype)
    torch.cuda.synchronize()
    with pytest.raises(pyreloc.TransferError) as e:
        mx.linear(x, q, dtype=dtype)
    assert e.value.code == "backend_failure"
    assert torch.equal(mx.linear(x, q, dtype=dtype), want)


@pytest.mark.gpu
def test_gate_gradient_in_a_feed_forward_layer_from_both_sides():
    """The gate's gradient from the 8-bit copies of what the first product
    gave, against 64 bits, too small as well as too large. bf16 results: half a
    step; 32-bit arithmetic in front of it: (16 + |g|) 2^-24 of the terms'
    size, 1 + g (1 - s) cancelling near its zero, as in test_silu_mul."""
    x = tensor((74, 128), torch.bfloat16, 82)
    weight = tensor((2 * 352, 128), torch.bfloat16, 83, 0.1)
    down = tensor((128, 352), torch.bfloat16, 84, 0.1)
    dy = tensor((74, 128), torch.bfloat16, 85)
    a = mx.linear(x, mx.quantize(weight)).detach().requires_grad_()
    got, = torch.autograd.grad(mx.linear(mx.silu_mul(a), down.requires_grad_()), a, dy)
    dh = host(mx.matmul(mx.quantize(dy), mx.quantize(down, along=0), dtype=torch.bfloat16))
    g, u = O.rounded(host(a)[:, :352], "mxint8"), O.rounded(host(a)[:, 352:], "mxint8")
    with np.errstate(over="ignore"):
        s = 1 / (1 + np.exp(-g))
    want = np.concatenate((dh * u * s * (1 + g * (1 - s)), dh * g * s), 1)
    size = np.concatenate((np.abs(dh * u) * s * (1 + np.abs(g) * (1 - s)), np.abs(dh * g * s)), 1)
    rel = (16 + np.abs(np.concatenate((g, g), 1))) * 2.0 ** -24 + 2.0 ** -22
    half = HALF_STEP[torch.bfloat16]
    # subnormal s: steps of 2^-149, as in test_silu_mul
    sub = 2.0 ** -147 * (2 + np.abs(np.concatenate((g, g), 1))) * (1 + np.concatenate((np.abs(dh * u), np.abs(dh)), 1))
    off = np.abs(host(got) - want) - (size * rel * (1 + half) + half * np.abs(want) + sub + 2.0 ** -126 * half)
    assert off.max() <= 0, off.max()
