"""Microscaled matrices: 4-bit weights and products, 8-bit activation checkpoints.

A row is cut into blocks of 32 values that share one power-of-two scale. Two
formats (exact definitions: the last section of ``include/sym_b200.h``):

``mxfp4``
    4-bit floating point (0, .5, 1, 1.5, 2, 3, 4, 6 with a sign), 4.25 bits per
    value: weights, and the operands of products on the tensor cores.
``mxint8``
    8-bit integers, 8.25 bits per value: activations kept for a backward pass.

They stand beside the int8 paths of this package: ``workloads.WeightFetcher``
expands int8 weights to ``[in, out]`` values, ``dequantize(w, transpose=True)``
does so for mxfp4 weights, and ``linear`` multiplies with them directly.

``quantize`` / ``quantize_both``   values -> codes, along the last axis or the first
``dequantize``                     codes -> values, in their layout or transposed
``matmul``                         product of two mxfp4 matrices
``linear``                         values times an mxfp4 weight (serving), or times a
                                   float weight with all three products of a training
                                   step on mxfp4 operands
``check``                          raises where a product did not complete
``silu_mul``                       silu(gate) * up, keeping gate and up in 8 bits for
                                   the backward pass

All calls run on the current stream of the tensors' device, allocate from
torch's caching allocator only and can be captured into CUDA graphs (a backward
pass, as torch asks, only while no eager graph of the same leaves is alive).
They have no CPU execution. Wrong arguments raise ``ValueError`` or ``TypeError``; failures of the
native layer raise ``pyreloc.TransferError``. A product's waits are bounded; one
that ran out is reported by the next product on its device, or by ``check``.

Derivatives are those of reverse mode, once; codes carry none. Forward-mode
tangents, ``vmap`` and second derivatives are refused. The kernels get addresses, which
a recorder of torch operations cannot see: ``make_fx`` is refused with
``NotImplementedError``, and so is ``torch.jit.trace`` but for ``linear`` and
``silu_mul``, which it records as autograd functions; ``torch.compile`` runs the
calls as they are, between its graphs.
"""
from __future__ import annotations

import ctypes
import operator
import threading
from functools import lru_cache

import torch
import torch.autograd.forward_ad as _forward_ad

from . import _native
from .pyreloc import _raise_transfer

BLOCK = 32
FORMATS = {"mxfp4": 0, "mxint8": 1}
_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_CODE_BYTES = {"mxfp4": 16, "mxint8": 32}  # per block


class _Scratch(threading.local):
    def __init__(self):
        self.error = _native.SbError()
        self.ref = ctypes.byref(self.error)


_scratch = _Scratch()


def _check(rc):
    if rc:
        _raise_transfer(_scratch.error)


def _stream(index):
    """The current stream (a cudaStream_t) of a device."""
    return torch._C._cuda_getCurrentRawStream(index)


_modes = torch._C._len_torch_dispatch_stack
_key_included = torch._C._dispatch_tls_is_dispatch_key_included
_PRE_DISPATCH = torch._C.DispatchKey.PreDispatch
_jit_tracing = torch._C._is_tracing
_compiling = torch.compiler.is_dynamo_compiling


def _uncompiled(call, *args, **kwargs):
    """A call as torch.compile runs it: as it is, between two graphs. Its frames
    are not taken apart, which would free tensors whose addresses a kernel is
    still to get."""
    return torch.compiler.disable(call)(*args, **kwargs)


def _traceable(call, jit=False):
    """Refuses a call whose result a recorder would keep as the allocation alone:
    under make_fx, and where the call is no autograd function (``jit``) under
    torch.jit.trace. Called where some dispatch mode or a tracer is at work."""
    from torch.fx.experimental.proxy_tensor import get_proxy_mode

    if get_proxy_mode() is not None:
        raise NotImplementedError(f"{call} cannot be recorded by make_fx: its kernels take addresses")
    if jit and _jit_tracing():
        raise NotImplementedError(f"{call} cannot be recorded by torch.jit.trace: its kernels take addresses")


def _no_tangents(call, *tensors):
    """Refuses inputs with forward-mode tangents, which would be lost."""
    for t in tensors:
        if isinstance(t, torch.Tensor) and _forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{call} has no forward-mode derivative")


_library = None


def _lib():
    global _library
    if _library is None:
        _library = _native.lib()
    return _library


def _blocks(cols):
    return -(-cols // BLOCK)


def _up256(n):
    return -(-n // 256) * 256


def _scale_bytes(rows, cols, format):
    if format == "mxfp4":
        return -(-rows // 128) * -(-cols // 128) * 512
    return rows * _blocks(cols)


class MxTensor:
    """A microscaled matrix ``[rows, cols]``: uint8 ``codes`` ``[rows, bytes]``
    and uint8 ``scales`` (flat, in the format's order).

    The constructor takes tensors that already have that layout, without a
    copy; ``from_rows`` takes row-major scales, as checkpoints hold them, and
    pads them. Products take 64 values of a row at a time and trust the padding:
    codes past a row's end are 0, and so are, in mxfp4's tiles, the scale bytes
    that a row's last tile has for blocks that do not exist (what it has for
    rows past the last is not read). Of tensors in host memory the constructor
    checks those bytes; on a device that would have to wait for the data, so what
    comes from elsewhere is best brought as host tensors or by ``from_rows``. A
    matrix keeps its tensors; they are not exchanged for others (``native``
    holds their addresses), but copies and pickles are made from them."""

    __slots__ = ("_codes", "_scales", "_shape", "_format", "_native")
    codes = property(lambda self: self._codes)
    scales = property(lambda self: self._scales)
    shape = property(lambda self: self._shape)
    format = property(lambda self: self._format)
    native = property(lambda self: self._native)

    def __init__(self, codes, scales, shape, format="mxfp4"):
        if format not in FORMATS:
            raise ValueError(f"format must be one of {sorted(FORMATS)}")
        rows, cols = map(operator.index, shape)
        if not isinstance(codes, torch.Tensor) or not isinstance(scales, torch.Tensor):
            raise TypeError("codes and scales are uint8 tensors")
        if rows < 0 or cols < 1:
            raise ValueError("a microscaled matrix has at least one column")
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise TypeError("codes and scales are uint8 tensors")
        on_cuda = codes.is_cuda
        if codes.get_device() != scales.get_device() or not on_cuda and codes.device != scales.device:
            raise ValueError("codes and scales live on different devices")
        blocks = _blocks(cols)
        width = blocks * _CODE_BYTES[format]
        if codes.shape != (rows, width) or not codes.is_contiguous():
            raise ValueError(f"{format} codes of [{rows}, {cols}] are a contiguous [{rows}, {width}] tensor")
        held = _scale_bytes(rows, cols, format)
        if scales.numel() != held or not scales.is_contiguous():
            raise ValueError(f"{format} scales of [{rows}, {cols}] are {held} contiguous bytes")
        self._codes, self._scales, self._shape, self._format = codes, scales, (rows, cols), format
        self._native = None
        if on_cuda and rows:
            at, scales_at = codes.data_ptr(), scales.data_ptr()
            if at % 16 or scales_at % 16:
                raise ValueError("codes and scales start on 16-byte boundaries")
            self._native = _native.SbMx(at, scales_at, rows, cols, FORMATS[format], codes.get_device())
        elif blocks % 4 and format == "mxfp4" and codes.device.type == "cpu":
            last = scales.view(-(-rows // 128), -(-blocks // 4), 32, 4, 4)[:, -1].transpose(1, 2)
            if last.reshape(-1, 4)[:rows, blocks % 4:].any():
                raise ValueError("scale bytes of blocks that do not exist are 0 in a row's last tile")

    @classmethod
    def _empty(cls, like, rows, cols, format="mxfp4"):
        """An uninitialised matrix on the device of ``like``."""
        q = cls.__new__(cls)
        q._codes = codes = like.new_empty((rows, _blocks(cols) * _CODE_BYTES[format]), dtype=torch.uint8)
        q._scales = scales = like.new_empty(_scale_bytes(rows, cols, format), dtype=torch.uint8)
        q._shape, q._format, q._native = (rows, cols), format, None
        if rows:
            q._native = _native.SbMx(codes.data_ptr(), scales.data_ptr(), rows, cols, FORMATS[format],
                                     like.get_device())
        return q

    def __reduce__(self):
        return MxTensor, (self._codes, self._scales, self._shape, self._format)

    @classmethod
    def from_rows(cls, codes, row_scales, cols, format="mxfp4"):
        """From codes and row-major scales ``[rows, blocks]``."""
        if not isinstance(codes, torch.Tensor) or not isinstance(row_scales, torch.Tensor):
            raise TypeError("codes and row_scales are uint8 tensors")
        cols = operator.index(cols)
        rows, blocks = row_scales.shape
        if blocks != _blocks(cols):
            raise ValueError(f"rows of {cols} values have {_blocks(cols)} scales")
        if format == "mxfp4":
            tiles = torch.nn.functional.pad(row_scales, (0, -blocks % 4, 0, -rows % 128))
            row_scales = tiles.view(-(-rows // 128), 4, 32, -(-blocks // 4), 4).permute(0, 3, 2, 1, 4)
        return cls(codes.contiguous(), row_scales.contiguous().flatten(), (rows, cols), format)

    def row_scales(self):
        """The scale bytes, row-major ``[rows, blocks]``."""
        rows, cols = self.shape
        blocks = _blocks(cols)
        if self.format == "mxint8":
            return self.scales.view(rows, blocks)
        tiles = self.scales.view(-(-rows // 128), -(-blocks // 4), 32, 4, 4).permute(0, 3, 2, 1, 4)
        return tiles.reshape(-(-rows // 128) * 128, -(-blocks // 4) * 4)[:rows, :blocks].contiguous()

    @property
    def device(self):
        return self._codes.device

    def get_device(self):
        return self._codes.get_device()

    def to(self, device, non_blocking=False):
        return MxTensor(self.codes.to(device, non_blocking=non_blocking),
                        self.scales.to(device, non_blocking=non_blocking), self.shape, self.format)

    def __repr__(self):
        return f"MxTensor({list(self.shape)}, {self.format}, {self.device})"


def _matrix(x, cols):
    """x [..., cols] as a matrix whose columns are adjacent: (tensor, rows, cols, row stride)."""
    if x.is_neg():  # a view whose memory holds the negated values
        x = x.resolve_neg()
    if x.is_contiguous():
        return x, x.numel() // cols, cols, cols
    if x.dim() != 2:
        x = x.reshape(-1, cols)
    rows = x.shape[0]
    if cols > 1 and x.stride(1) != 1:
        x = x.contiguous()
    return x, rows, cols, x.stride(0) if rows > 1 else cols


def _values(x, name):
    """The shape of a tensor of values, once it is one that the kernels take."""
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name} is a tensor")
    if x.dtype not in _DTYPES:
        raise TypeError(f"{name} is float32, float16 or bfloat16")
    if not x.is_cuda:
        raise ValueError(f"{name} is on {x.device}: microscaled operators run on CUDA devices")
    shape = x.shape
    if not shape or shape[-1] == 0:
        raise ValueError(f"{name} needs at least one column")
    return shape


def _mx(q, name, format=None):
    if type(q) is not MxTensor:
        raise TypeError(f"{name} is an MxTensor")
    if not q._codes.is_cuda:
        raise ValueError(f"{name} is on {q.device}: microscaled operators run on CUDA devices")
    if format is not None and q._format != format:
        raise ValueError(f"{name} is {q._format}: {format} is needed")
    return q


def _result(dtype):
    if dtype not in _DTYPES:
        raise TypeError("results are float32, float16 or bfloat16")
    return dtype


def _quantize(x, cols, format, along, across):
    x, rows, cols, stride = _matrix(x, cols)
    q = MxTensor._empty(x, rows, cols, format) if along else None
    qt = MxTensor._empty(x, cols, rows) if across else None
    if rows:
        _check(_lib().sb_mx_quantize(x.data_ptr(), _DTYPES[x.dtype], rows, cols, stride, q.native if along else None,
                                     qt.native if across else None, _stream(x.get_device()), _scratch.ref))
    return q, qt


@lru_cache(maxsize=4096)
def _layout(*matrices):
    """Several microscaled matrices ((rows, cols, format) each, or None) in one
    buffer, for what lives no longer than a call or is kept for one backward
    pass: one allocation, and one tensor to keep. -> its size and the places."""
    at, places = 0, []
    for m in matrices:
        if m is None:
            places.append(None)
            continue
        rows, cols, format = m
        scales = at + _up256(rows * _blocks(cols) * _CODE_BYTES[format])
        places.append((at, scales, rows, cols, FORMATS[format]))
        at = scales + _up256(_scale_bytes(rows, cols, format))
    return at, tuple(places)


def _placed(buffer, places):
    """Descriptors of the matrices of a ``_layout`` in its buffer."""
    base, index = buffer.data_ptr(), buffer.get_device()
    return [None if p is None else _native.SbMx(base + p[0], base + p[1], p[2], p[3], p[4], index) for p in places]


def _differentiable_once(backward):
    """torch's once_differentiable, whose wrapping is only paid for where a
    graph of the backward pass is asked for."""
    guarded = torch.autograd.function.once_differentiable(backward)

    def run(ctx, *grads):
        if _compiling():
            return _uncompiled(run, ctx, *grads)
        if _modes() or _key_included(_PRE_DISPATCH):
            _traceable("a backward pass")
        if _forward_ad._current_level >= 0:
            _no_tangents("a backward pass", *grads)
        return (guarded if torch.is_grad_enabled() else backward)(ctx, *grads)

    return run


def _quantize_into(x, along, across):
    x, rows, cols, stride = _matrix(x, x.shape[-1])
    _check(_lib().sb_mx_quantize(x.data_ptr(), _DTYPES[x.dtype], rows, cols, stride, along, across,
                                 _stream(x.get_device()), _scratch.ref))


def _matmul_into(a, b, y):
    _check(_lib().sb_mx_matmul(a, b, y.data_ptr(), _DTYPES[y.dtype], _stream(y.get_device()), _scratch.ref))
    return y


def quantize(x, format="mxfp4", *, along=-1):
    """Values ``[..., cols]`` to an ``MxTensor`` ``[rows, cols]`` whose blocks run
    along the last axis (leading axes are flattened), or for a matrix with
    ``along=0`` to the mxfp4 form of its transpose, whose blocks run along
    the first axis."""
    if _compiling():
        return _uncompiled(quantize, x, format, along=along)
    if _modes() or _key_included(_PRE_DISPATCH) or _jit_tracing():
        _traceable("quantize", jit=True)
    shape = _values(x, "x")
    if format not in FORMATS:
        raise ValueError(f"format must be one of {sorted(FORMATS)}")
    if along not in (0, -1):
        raise ValueError("along must be -1 or 0")
    if along == 0:
        if len(shape) != 2 or shape[0] == 0:
            raise ValueError("along=0 takes a matrix with at least one row")
        if format != "mxfp4":
            raise ValueError("along=0 is defined for mxfp4")
    if len(shape) == 2 and format == "mxfp4" and shape[0] > 1 and shape[1] > 1 and x.stride(0) == 1 != x.stride(1):
        # a transposed view: the other direction of the matrix behind it
        return _quantize(x.t(), shape[0], format, along == 0, along != 0)[0 if along == 0 else 1]
    q, qt = _quantize(x, shape[-1], format, along != 0, along == 0)
    return q if qt is None else qt


def quantize_both(x):
    """A matrix's two mxfp4 forms with one read of it: ``(quantize(x),
    quantize(x, along=0))``, what a training step's products take."""
    if _compiling():
        return _uncompiled(quantize_both, x)
    if _modes() or _key_included(_PRE_DISPATCH) or _jit_tracing():
        _traceable("quantize_both", jit=True)
    shape = _values(x, "x")
    if len(shape) != 2 or shape[0] == 0:
        raise ValueError("quantize_both takes a matrix with at least one row")
    return _quantize(x, shape[1], "mxfp4", True, True)


def dequantize(q, dtype=torch.float16, *, transpose=False):
    """The values of an ``MxTensor``, each rounded once to ``dtype``: ``[rows,
    cols]``, or ``[cols, rows]`` with ``transpose`` (mxfp4), the layout that a
    product ``x @ w`` takes."""
    if _compiling():
        return _uncompiled(dequantize, q, dtype, transpose=transpose)
    if _modes() or _key_included(_PRE_DISPATCH) or _jit_tracing():
        _traceable("dequantize", jit=True)
    _mx(q, "q")
    dtype = _result(dtype)
    if transpose and q.format != "mxfp4":
        raise ValueError("transpose is defined for mxfp4")
    rows, cols = q.shape
    out = q._codes.new_empty((cols, rows) if transpose else (rows, cols), dtype=dtype)
    if rows:
        _check(_lib().sb_mx_dequantize(q.native, out.data_ptr(), _DTYPES[dtype], int(transpose),
                                       _stream(q.get_device()), _scratch.ref))
    return out


@lru_cache(maxsize=4096)
def _linear_workspace(m, n, k, device):
    size = ctypes.c_int64()
    _check(_lib().sb_mx_linear_workspace(m, n, k, device, ctypes.byref(size), _scratch.ref))
    return size.value


def matmul(a, b, *, dtype=torch.bfloat16):
    """``a [m, k]`` times the transpose of ``b [n, k]``, both mxfp4, accumulated in
    32 bits and rounded once to ``dtype``."""
    if _compiling():
        return _uncompiled(matmul, a, b, dtype=dtype)
    if _modes() or _key_included(_PRE_DISPATCH) or _jit_tracing():
        _traceable("matmul", jit=True)
    _mx(a, "a", "mxfp4"), _mx(b, "b", "mxfp4")
    dtype = _result(dtype)
    if a.get_device() != b.get_device():
        raise ValueError("a and b live on different devices")
    (m, k), (n, kb) = a.shape, b.shape
    if k != kb:
        raise ValueError(f"a [m, k] and b [n, k] need the same k: got {k} and {kb}")
    y = a._codes.new_empty((m, n), dtype=dtype)
    return _matmul_into(a.native, b.native, y) if m and n else y


def check(device=None):
    """Waits for the work of a device (default: the current one) and raises
    ``pyreloc.TransferError`` where a product's bounded wait ran out since the
    last report, so that its result is incomplete. The next eager product on the
    device reports it too; this call is for those that none follows, replays of
    captured graphs among them."""
    if device is None or isinstance(device, int):
        index = device
    else:
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError(f"microscaled operators run on CUDA devices: got {device}")
        index = device.index
    if index is None:
        index = torch.cuda.current_device()
    torch.cuda.synchronize(index)
    _check(_lib().sb_mx_status(index, _scratch.ref))


def _linear(x, w, dtype, shape):
    """x [shape] times the transpose of w."""
    n, k = w._shape
    x, m, _, stride = _matrix(x, k)
    y = x.new_empty((*shape[:-1], n), dtype=dtype)
    if m and n:
        index = x.get_device()
        size = _linear_workspace(m, n, k, index)
        space = x.new_empty(size, dtype=torch.uint8) if size else None
        _check(_lib().sb_mx_linear(x.data_ptr(), _DTYPES[x.dtype], m, stride, w._native, y.data_ptr(), _DTYPES[dtype],
                                   space.data_ptr() if size else None, size, _stream(index), _scratch.ref))
    return y


class _FrozenLinear(torch.autograd.Function):
    """A product with a 4-bit weight that is not trained."""

    @staticmethod
    def forward(ctx, x, w, wt, dtype):
        ctx.shape = None
        if wt is not None:
            ctx.save_for_backward(wt.codes, wt.scales)
            ctx.shape, ctx.dtype = wt.shape, x.dtype
        return _linear(x, w, dtype, x.shape)

    @staticmethod
    @_differentiable_once
    def backward(ctx, dy):
        if ctx.shape is None:
            raise ValueError("x needs a gradient: linear was recorded without weight_t")
        return _linear(dy, MxTensor(*ctx.saved_tensors, ctx.shape), ctx.dtype, dy.shape), None, None, None


class _TrainLinear(torch.autograd.Function):
    """y = Q(x) Q(w)^T, dx = Q(dy) Q(w^T)^T, dw = Q(dy^T) Q(x^T)^T; every
    tensor is read once for the forms that it is needed in, and what is kept
    for the backward pass is kept in 4 bits."""

    @staticmethod
    def forward(ctx, x, weight, dtype):
        need_x, need_w, _ = ctx.needs_input_grad
        n, k = weight.shape
        m = x.numel() // k
        ctx.dtypes, ctx.shape, ctx.extents = (x.dtype, weight.dtype), x.shape, (m, n, k)
        if m == 0 or n == 0:  # no rows, or no columns of the result: gradients of zeros
            return x.new_empty((*x.shape[:-1], n), dtype=dtype)
        size, places = _layout((m, k, "mxfp4"), (n, k, "mxfp4"))
        now = x.new_empty(size, dtype=torch.uint8)
        qx, qw = _placed(now, places)
        size, ctx.places = _layout((k, m, "mxfp4") if need_w else None, (k, n, "mxfp4") if need_x else None)
        kept = x.new_empty(size, dtype=torch.uint8)
        qxt, qwt = _placed(kept, ctx.places)
        ctx.save_for_backward(kept)
        _quantize_into(x, qx, qxt)
        _quantize_into(weight, qw, qwt)
        return _matmul_into(qx, qw, x.new_empty((*x.shape[:-1], n), dtype=dtype))

    @staticmethod
    @_differentiable_once
    def backward(ctx, dy):
        need_x, need_w, _ = ctx.needs_input_grad
        m, n, k = ctx.extents
        if m == 0 or n == 0:
            return (dy.new_zeros(ctx.shape, dtype=ctx.dtypes[0]) if need_x else None,
                    dy.new_zeros((n, k), dtype=ctx.dtypes[1]) if need_w else None, None)
        kept, = ctx.saved_tensors
        qxt, qwt = _placed(kept, ctx.places)
        size, places = _layout((m, n, "mxfp4") if need_x else None, (n, m, "mxfp4") if need_w else None)
        now = dy.new_empty(size, dtype=torch.uint8)
        qdy, qdyt = _placed(now, places)
        _quantize_into(dy, qdy, qdyt)
        dx = _matmul_into(qdy, qwt, dy.new_empty(ctx.shape, dtype=ctx.dtypes[0])) if need_x else None
        dw = _matmul_into(qdyt, qxt, dy.new_empty((n, k), dtype=ctx.dtypes[1])) if need_w else None
        return dx, dw, None


def linear(x, weight, weight_t=None, *, dtype=None):
    """``x [..., k]`` times the transpose of ``weight [n, k]``, with both operands in
    mxfp4 (blocks along k) and 32-bit accumulation; the result ``[..., n]`` has
    ``dtype`` (default: that of x).

    ``weight`` an ``MxTensor``: serving, any number of rows of x from one token
    up. x is quantised in the call. Where x needs a gradient, pass
    ``weight_t``, the mxfp4 form of the weight's transpose (``quantize_both``), for
    ``dx = Q(dy) weight_t^T``.

    ``weight`` a float tensor: training; x, weight and dy are quantised along the
    axis that each product sums over, and the backward pass gives dx and dw.
    Where no gradient is asked for, the forms along k are made and dropped."""
    if _compiling():
        return _uncompiled(linear, x, weight, weight_t, dtype=dtype)
    if _modes() or _key_included(_PRE_DISPATCH):
        _traceable("linear")
    if _forward_ad._current_level >= 0:
        _no_tangents("linear", x, weight)
    shape = _values(x, "x")
    dtype = x.dtype if dtype is None else _result(dtype)
    frozen = type(weight) is MxTensor
    if frozen:
        n, k = _mx(weight, "weight", "mxfp4")._shape
    elif weight_t is not None:
        raise ValueError("weight_t goes with an MxTensor weight")
    else:
        extents = _values(weight, "weight")
        if len(extents) != 2:
            raise ValueError("weight is a matrix [n, k]")
        n, k = extents
    if weight.get_device() != x.get_device():
        raise ValueError("x and weight live on different devices")
    if shape[-1] != k:
        raise ValueError(f"x [..., k] and weight [n, k] need the same k: got {shape[-1]} and {k}")
    if frozen:
        needs = x.requires_grad and torch.is_grad_enabled()
        if not (needs or _jit_tracing()):
            return _linear(x, weight, dtype, shape)
        if weight_t is None:
            if not needs:
                return _FrozenLinear.apply(x, weight, None, dtype)
            raise ValueError("x needs a gradient: pass weight_t, the mxfp4 form of the weight's transpose")
        if _mx(weight_t, "weight_t", "mxfp4").shape != (k, n) or weight_t.device != x.device:
            raise ValueError(f"weight_t is [{k}, {n}] on {x.device}")
        return _FrozenLinear.apply(x, weight, weight_t, dtype)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad) or _jit_tracing():
        return _TrainLinear.apply(x, weight, dtype)
    # nothing to keep for a backward pass: the forms along k alone
    return _linear(x, _quantize(weight, k, "mxfp4", True, False)[0], dtype, shape)


class _SiluMul(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate, up):
        ctx.packed, ctx.shape = up is None, gate.shape
        if up is None:
            gate, up = gate.chunk(2, -1)
        cols = gate.shape[-1]
        kept_matrix = (gate.numel() // cols, cols, "mxint8")
        size, ctx.places = _layout(kept_matrix, kept_matrix)
        kept = gate.new_empty(size, dtype=torch.uint8)
        ctx.save_for_backward(kept)
        return _silu_mul(gate, up, *_placed(kept, ctx.places))

    @staticmethod
    @_differentiable_once
    def backward(ctx, dh):
        kept, = ctx.saved_tensors
        gate, up = _placed(kept, ctx.places)
        dgate = dh.new_empty(ctx.shape)
        dup = None if ctx.packed else dh.new_empty(ctx.shape)
        if gate.rows:
            cols, dtype = gate.cols, dh.dtype
            dh, _, _, stride = _matrix(dh, cols)
            out = 2 * cols if ctx.packed else cols
            at = dgate.data_ptr() + cols * dh.element_size() if ctx.packed else dup.data_ptr()
            _check(_lib().sb_silu_mul_backward(dh.data_ptr(), stride, _DTYPES[dtype], gate, up, dgate.data_ptr(), out,
                                               at, out, _stream(dh.get_device()), _scratch.ref))
        return dgate, dup


def _silu_mul(gate, up, kept_gate=None, kept_up=None):
    shape = gate.shape
    h = gate.new_empty(shape)
    gate, rows, cols, gate_stride = _matrix(gate, shape[-1])
    up, _, _, up_stride = _matrix(up, cols)
    if rows:
        index = gate.get_device()
        _check(_lib().sb_silu_mul(gate.data_ptr(), gate_stride, up.data_ptr(), up_stride, _DTYPES[gate.dtype], rows,
                                  cols, index, h.data_ptr(), kept_gate, kept_up, _stream(index), _scratch.ref))
    return h


def silu_mul(gate, up=None):
    """``silu(gate) * up`` elementwise, ``silu(g) = g / (1 + exp(-g))``; with ``up``
    left out, ``gate`` holds both halves along its last axis.

    Where a gradient is needed, gate and up are kept as mxint8 copies (8.25 bits
    per value, step at most 2^-6 of the block's largest magnitude) instead of
    as they are, and the backward pass computes both gradients from the copies.
    The result itself is computed from the inputs."""
    if _compiling():
        return _uncompiled(silu_mul, gate, up)
    if _modes() or _key_included(_PRE_DISPATCH):
        _traceable("silu_mul")
    if _forward_ad._current_level >= 0:
        _no_tangents("silu_mul", gate, up)
    shape = _values(gate, "gate")
    if up is None:
        if shape[-1] % 2:
            raise ValueError("gate and up in one tensor need an even last axis")
    else:
        if _values(up, "up") != shape or up.dtype != gate.dtype or up.device != gate.device:
            raise ValueError("gate and up have the same shape, type and device")
    needs = torch.is_grad_enabled() and (gate.requires_grad or (up is not None and up.requires_grad))
    if needs or _jit_tracing():
        return _SiluMul.apply(gate, up)
    return _silu_mul(*gate.chunk(2, -1)) if up is None else _silu_mul(gate, up)
