"""The bytes of a quantised matrix are those of its values alone: nothing of
the memory's past is left in them."""
import mx_oracle as O
import numpy as np
import pytest
import torch
from test_microscale_gpu import host, tensor

from sym_b200 import microscale as mx

pytestmark = pytest.mark.gpu


def dirty():
    """Leaves 0xa5 in the allocator's free memory."""
    for size in (1 << 9, 1 << 12, 1 << 16, 1 << 19, 1 << 22, 1 << 24):
        held = [torch.full((size,), 0xA5, dtype=torch.uint8, device="cuda") for _ in range(4)]
        del held


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 4096), (3, 40), (31, 129), (33, 32), (127, 260), (128, 96), (129, 129),
                                       (200, 1000), (257, 500), (1000, 4100), (4097, 1030), (2500, 8191)])
def test_every_byte_of_the_scales_is_defined(rows, cols, dtype):
    x = tensor((rows, cols), dtype, rows)
    for view in (x, tensor((rows, cols + 3), dtype, rows)[:, 3:]):
        want, across = (O.tile_scales(O.quantize(v, "mxfp4")[1]) for v in (host(view), host(view).T))
        dirty()
        q, qt = mx.quantize_both(view)
        dirty()
        q1 = mx.quantize(view)
        dirty()
        q0 = mx.quantize(view, along=0)
        for got, oracle in ((q, want), (q1, want), (qt, across), (q0, across)):
            assert np.array_equal(got.scales.cpu().numpy(), oracle)
        assert torch.equal(q.codes, q1.codes) and torch.equal(qt.codes, q0.codes)


def test_matrices_behind_and_before_stay_as_they_were():
    """Through the C call, into the middle of a buffer: whole tiles are
    written, nothing beside them."""
    import ctypes

    from sym_b200 import _native

    rows, cols = 130, 200
    x = tensor((rows, cols), torch.float16, 1)
    scale_bytes = 2 * 2 * 512
    buffers = [torch.full((1024 + n + 1024,), 0xA5, dtype=torch.uint8, device="cuda")
               for n in (rows * 7 * 16, scale_bytes, cols * 5 * 16, scale_bytes)]
    at = [b.data_ptr() + 1024 for b in buffers]
    along = _native.SbMx(at[0], at[1], rows, cols, 0, 0)
    across = _native.SbMx(at[2], at[3], cols, rows, 0, 0)
    err = _native.SbError()
    stream = torch.cuda.current_stream().cuda_stream
    assert _native.lib().sb_mx_quantize(x.data_ptr(), 1, rows, cols, cols, along, across, stream, ctypes.byref(err)) == 0
    torch.cuda.synchronize()
    for b in buffers:
        assert (b[:1024] == 0xA5).all() and (b[-1024:] == 0xA5).all()
    for b, v in ((buffers[1], host(x)), (buffers[3], host(x).T)):
        assert np.array_equal(b[1024:-1024].cpu().numpy(), O.tile_scales(O.quantize(v, "mxfp4")[1]))
