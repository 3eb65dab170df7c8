"""Matrices brought in tile order: the padding that products trust is checked
where that needs no waiting, and what they do not read changes nothing."""
import pytest
import torch

from sym_b200 import microscale as mx

SHAPES = [(1, 1), (3, 40), (128, 96), (130, 260), (257, 500), (5, 4110)]


def tiles_of(q):
    """q's scales as [rows of whole tiles, blocks of whole tiles]: a copy, and how to put one back."""
    rows, cols = q.shape
    tr, tq = -(-rows // 128), -(-cols // 128)
    flat = q.scales.view(tr, tq, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(tr * 128, tq * 4).clone()
    return flat, lambda f: f.view(tr, 4, 32, tq, 4).permute(0, 3, 2, 1, 4).flatten()


def matrix(rows, cols):
    g = torch.Generator().manual_seed(rows)
    codes = torch.randint(0, 256, (rows, -(-cols // 32) * 16), generator=g, dtype=torch.uint8)
    scales = torch.randint(100, 140, (rows, -(-cols // 32)), generator=g, dtype=torch.uint8)
    return mx.MxTensor.from_rows(codes, scales, cols)


@pytest.mark.parametrize("rows,cols", SHAPES)
def test_scales_of_blocks_that_do_not_exist_are_refused(rows, cols):
    q = matrix(rows, cols)
    blocks = -(-cols // 32)
    flat, back = tiles_of(q)
    assert torch.equal(back(flat), q.scales)
    if blocks % 4 == 0:
        mx.MxTensor(q.codes, q.scales, q.shape)
        return
    for r in {0, rows // 2, rows - 1}:
        for b in range(blocks, flat.shape[1]):
            for byte in (1, 255):
                bad = flat.clone()
                bad[r, b] = byte
                with pytest.raises(ValueError, match="do not exist"):
                    mx.MxTensor(q.codes, back(bad), q.shape)
    # rows past the last are nobody's
    flat[rows:] = 255
    assert mx.MxTensor(q.codes, back(flat), q.shape).shape == q.shape
    mx.MxTensor(torch.zeros(0, blocks * 16, dtype=torch.uint8), torch.zeros(0, dtype=torch.uint8), (0, cols))


def test_what_is_no_matrix_is_refused_as_such():
    codes, scales, rows = (torch.zeros(*s, dtype=torch.uint8) for s in ((4, 32), (512,), (4, 2)))
    for call in (lambda: mx.MxTensor(None, scales, (4, 64)), lambda: mx.MxTensor(codes, [0] * 512, (4, 64)),
                 lambda: mx.MxTensor(codes, scales, (4.0, 64)), lambda: mx.MxTensor(codes, scales, (4, "64")),
                 lambda: mx.MxTensor(codes, scales, 256), lambda: mx.MxTensor.from_rows(None, rows, 64),
                 lambda: mx.MxTensor.from_rows(codes, [[0, 0]] * 4, 64), lambda: mx.MxTensor.from_rows(codes, rows, 64.0)):
        with pytest.raises(TypeError):
            call()
    for call in (lambda: mx.MxTensor(codes, scales, (4,)), lambda: mx.MxTensor(codes, scales, (4, 64, 1)),
                 lambda: mx.MxTensor.from_rows(codes, rows[0], 64), lambda: mx.MxTensor.from_rows(codes, rows, 0),
                 lambda: mx.MxTensor.from_rows(codes, rows, 64, "fp4")):
        with pytest.raises(ValueError):
            call()
    q = mx.MxTensor.from_rows(codes, rows, torch.tensor(64))
    assert q.shape == (4, 64) and all(type(n) is int for n in q.shape)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(1, 300, 2050), (8, 2000, 4110), (13, 20000, 65), (50, 19001, 70), (100, 300, 800),
                                   (180, 300, 4110), (163, 768, 130), (777, 11009, 2080), (1347, 9703, 66)])
def test_scales_of_rows_that_do_not_exist_change_nothing(m, n, k):
    g = torch.Generator().manual_seed(m)
    x, w = torch.randn(m, k, generator=g).cuda(), torch.randn(n, k, generator=g).cuda()
    matrices = [mx.quantize(x), mx.quantize(w)]
    want = mx.linear(x, matrices[1])
    other = []
    for q in matrices:
        flat, back = tiles_of(q)
        flat[q.shape[0]:] = 255
        other.append(mx.MxTensor(q.codes, back(flat), q.shape))
    assert want.isfinite().all()
    assert torch.equal(mx.linear(x, other[1]), want)
    assert torch.equal(mx.matmul(*other, dtype=x.dtype), want)
    for transpose in (False, True):
        assert torch.equal(mx.dequantize(other[1], transpose=transpose), mx.dequantize(matrices[1], transpose=transpose))
    # a block that exists and is marked keeps its meaning
    marked = matrices[1].row_scales()
    marked[:, -1] = 255
    assert mx.linear(x, mx.MxTensor.from_rows(matrices[1].codes, marked, k)).isnan().all()
