"""Microscaled matrices without a GPU: the formats' oracle against hand-made
values, the scale layout, and what the calls refuse."""
import ctypes
import math

import mx_oracle as O
import numpy as np
import pytest
import torch

from sym_b200 import _native
from sym_b200 import microscale as mx


def test_oracle_on_hand_made_blocks():
    x = np.zeros((1, 64))
    # largest 7 = 1.75 2^2: scale 2^0; ties to even codes, 7 saturates
    x[0, :12] = [7, 5, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, -5, -0.25, 0.26, 4.9]
    x[0, 32:35] = [2.0 ** -127, 2.0 ** -128, 2.0 ** -140]
    v = O.rounded(x)
    assert v[0, :12].tolist() == [6, 4, 0, 1, 1, 2, 2, 4, -4, 0, 0.5, 4]
    # scale clamped at 2^-127: 2^-128 is half of it, 2^-140 rounds to 0
    assert v[0, 32:35].tolist() == [2.0 ** -127, 2.0 ** -128, 0]
    q, s = O.quantize(x, "mxint8")
    assert s[0].tolist() == [2 + 127, 7]
    assert q[0, 0, :3].tolist() == [112, 80, 4]
    x[0, 3] = math.inf
    assert O.quantize(x, "mxfp4")[1][0].tolist() == [255, 0]
    assert np.isnan(O.rounded(x)[0, :32]).all() and not np.isnan(O.rounded(x)[0, 32:]).any()


@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 40), (128, 128), (130, 129), (257, 500)])
def test_scale_layout(rows, cols):
    rng = np.random.default_rng(rows)
    scale = rng.integers(0, 255, (rows, O.blocks_of(cols)), dtype=np.uint8)
    codes = torch.from_numpy(rng.integers(0, 255, (rows, O.blocks_of(cols) * 16), dtype=np.uint8))
    q = mx.MxTensor.from_rows(codes, torch.from_numpy(scale), cols)
    assert np.array_equal(q.scales.numpy(), O.tile_scales(scale))
    assert np.array_equal(q.row_scales().numpy(), scale)
    assert q.shape == (rows, cols) and q.to("cpu").format == "mxfp4"


def test_matrix_refusals():
    codes = torch.zeros(4, 32, dtype=torch.uint8)
    scales = torch.zeros(512, dtype=torch.uint8)
    mx.MxTensor(codes, scales, (4, 64))
    for bad in (dict(format="mxfp6"), dict(shape=(4, 32)), dict(shape=(4, 65)), dict(shape=(3, 64)),
                dict(shape=(4, 0)), dict(codes=torch.zeros(32, 4, dtype=torch.uint8).t()),
                dict(scales=scales[:-1]), dict(scales=torch.zeros(1024, dtype=torch.uint8)[::2]),
                dict(format="mxint8")):
        args = dict(codes=codes, scales=scales, shape=(4, 64), format="mxfp4") | bad
        with pytest.raises(ValueError):
            mx.MxTensor(**args)
    with pytest.raises(TypeError):
        mx.MxTensor(codes.float(), scales, (4, 64))
    with pytest.raises(ValueError):
        mx.MxTensor.from_rows(codes, torch.zeros(4, 3, dtype=torch.uint8), 64)


def test_calls_refuse_host_tensors_and_wrong_types():
    x = torch.zeros(4, 64)
    q = mx.MxTensor(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(512, dtype=torch.uint8), (4, 64))
    for call in (lambda: mx.quantize(x), lambda: mx.quantize_both(x), lambda: mx.dequantize(q),
                 lambda: mx.matmul(q, q), lambda: mx.linear(x, q), lambda: mx.linear(x, x), lambda: mx.silu_mul(x, x)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    for call in (lambda: mx.quantize(x.double()), lambda: mx.quantize([1.0]), lambda: mx.matmul(x, q),
                 lambda: mx.dequantize(x), lambda: mx.silu_mul(x.int(), x)):
        with pytest.raises(TypeError):
            call()


def _native_call(name, *args):
    err = _native.SbError()
    rc = getattr(_native.lib(), name)(*args, ctypes.byref(err))
    return rc, _native.error_of(err)[0]


def test_native_calls_refuse_before_they_launch():
    """Bad descriptors are answered with an error code before any CUDA call:
    these run without a device."""
    def q(**kw):
        a = dict(codes=4096, scales=8192, rows=4, cols=64, format=0, device=0) | kw
        return _native.SbMx(*(a[f] for f, _ in _native.SbMx._fields_))

    good = q()
    for bad in (q(codes=0), q(codes=4100), q(scales=8), q(rows=0), q(cols=-1), q(format=7), q(device=-1),
                q(rows=1 << 41), q(rows=1 << 39, cols=1 << 39)):
        assert _native_call("sb_mx_dequantize", bad, 4096, 0, 0, None) == (1, "invalid_view")
        assert _native_call("sb_mx_matmul", good, bad, 4096, 0, None) == (1, "invalid_view")
        assert _native_call("sb_mx_linear", 4096, 0, 1, 64, bad, 4096, 0, 4096, 1 << 40, None) == (1, "invalid_view")
        assert _native_call("sb_mx_quantize", 4096, 0, 4, 64, 64, bad, None, None) == (1, "invalid_view")
    assert _native_call("sb_mx_dequantize", None, 4096, 0, 0, None) == (1, "invalid_view")
    assert _native_call("sb_mx_dequantize", good, None, 0, 0, None) == (1, "invalid_view")
    assert _native_call("sb_mx_dequantize", good, 4096, 3, 0, None) == (1, "typed_unsupported")
    assert _native_call("sb_mx_dequantize", q(format=1), 4096, 0, 1, None) == (1, "typed_unsupported")
    assert _native_call("sb_mx_matmul", good, q(cols=32), 4096, 0, None) == (1, "invalid_view")
    assert _native_call("sb_mx_matmul", good, q(device=1), 4096, 0, None) == (1, "device_mismatch")
    assert _native_call("sb_mx_matmul", q(format=1), good, 4096, 0, None) == (1, "typed_unsupported")
    assert _native_call("sb_mx_quantize", 4096, 0, 4, 64, 64, None, None, None) == (1, "invalid_options")
    assert _native_call("sb_mx_quantize", 4096, 0, 5, 64, 64, good, None, None) == (1, "invalid_view")
    assert _native_call("sb_mx_quantize", 4096, 0, 4, 64, -1, good, None, None) == (1, "invalid_view")
    assert _native_call("sb_mx_quantize", 4096, 9, 4, 64, 64, good, None, None) == (1, "typed_unsupported")
    assert _native_call("sb_mx_quantize", 4096, 0, 64, 5, 5, None, good, None) == (1, "invalid_view")
    k = q(format=1)
    assert _native_call("sb_silu_mul", 4096, 64, 4096, 64, 0, 4, 64, 0, 4096, k, None, None) == (1, "invalid_options")
    assert _native_call("sb_silu_mul", 4096, 64, 4096, 64, 0, 4, 64, 0, 4096, k, good, None) == (1, "invalid_view")
    assert _native_call("sb_silu_mul", None, 64, 4096, 64, 0, 4, 64, 0, 4096, None, None, None) == (1, "invalid_view")
    assert _native_call("sb_silu_mul_backward", 4096, 64, 0, k, good, 4096, 64, 4096, 64, None) == (1, "invalid_view")
    assert _native_call("sb_silu_mul_backward", 4096, 64, 0, k, k, 4096, 63, 4096, 64, None) == (1, "invalid_view")
