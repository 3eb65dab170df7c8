"""Microscaled operators on the GPU against their definition in 64 bits.

Tolerances. Codes, scales and expanded values are exact: a power-of-two scale
leaves one rounding, whose result the definition fixes. A product's terms are
exact in 32 bits (two 2-bit significands), so its sum of K terms in any order,
each step off by at most one unit in the last place (2^-23), is off by at most
K 2^-23 sum |a b|; then one rounding to the result's type (half a step)."""
import mx_oracle as O
import numpy as np
import pytest
import torch

from sym_b200 import microscale as mx

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SHAPES = [(1, 1), (1, 32), (3, 31), (2, 33), (16, 8), (127, 129), (128, 128), (129, 260), (1, 4096), (300, 1000),
          (257, 7), (33, 2048)]


def tensor(shape, dtype, seed=0, std=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g) * std
    if x.numel() > 64:
        x.view(-1)[::17] *= 30
        x.view(-1)[5::29] = 0
    return x.to(dtype).cuda()


def host(x):
    return x.detach().double().cpu().numpy()


def stored(q):
    return q.codes.cpu().numpy(), q.row_scales().cpu().numpy()


def check_quantized(q, x, fmt="mxfp4"):
    want, scale = O.quantize(x, fmt)
    codes, got_scale = stored(q)
    assert q.shape == x.shape
    assert np.array_equal(got_scale, scale)
    assert np.array_equal(codes, O.code_bytes(want, fmt))
    if fmt == "mxfp4":  # bytes of the last tile past the row's end are 0, so that absent blocks add nothing
        tiles = q.scales.cpu().numpy()
        mine = O.tile_scales(scale)
        rows = x.shape[0]
        if rows % 128 == 0:
            assert np.array_equal(tiles, mine)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_quantize(shape, name):
    x = tensor(shape, TYPES[name], seed=shape[1])
    check_quantized(mx.quantize(x), host(x))
    check_quantized(mx.quantize(x, "mxint8"), host(x), "mxint8")
    check_quantized(mx.quantize(x, along=0), host(x).T)
    q, qt = mx.quantize_both(x)
    check_quantized(q, host(x))
    check_quantized(qt, host(x).T)


@pytest.mark.parametrize("name", TYPES)
def test_quantize_extreme_values(name):
    t = TYPES[name]
    big, tiny = torch.finfo(t).max, torch.finfo(t).smallest_normal
    sub = tiny * 2.0 ** -7
    rows = [torch.zeros(64), torch.full((64,), big), torch.full((64,), -big), torch.full((64,), sub),
            torch.linspace(-7, 7, 64), torch.arange(64) * sub, torch.full((64,), tiny)]
    for bad in (float("inf"), float("-inf"), float("nan")):
        r = torch.linspace(-1, 1, 64)
        r[40] = bad
        rows.append(r)
    x = torch.stack([r.to(t) for r in rows]).cuda()
    with np.errstate(invalid="ignore"):
        check_quantized(mx.quantize(x), host(x))
        check_quantized(mx.quantize(x, "mxint8"), host(x), "mxint8")
        check_quantized(mx.quantize(x, along=0), host(x).T)
    v = mx.dequantize(mx.quantize(x), torch.float32)
    assert torch.isnan(v[-3:, 32:]).all() and not torch.isnan(v[:, :32]).any()


def test_every_16_bit_pattern():
    bits = torch.arange(-(1 << 15), 1 << 15, dtype=torch.int16)
    for t in (torch.float16, torch.bfloat16):
        x = bits.view(t)
        x = torch.where(torch.isfinite(x), x, torch.zeros_like(x)).view(-1, 64).cuda()
        check_quantized(mx.quantize(x), host(x))
        check_quantized(mx.quantize(x, "mxint8"), host(x), "mxint8")


@pytest.mark.parametrize("name", TYPES)
def test_strides(name):
    t = TYPES[name]
    base = tensor((70, 300), t)
    for view in (base[:, :96], base[:, 3:100], base[::2], base[5:6], base[:, 1:2], base.t(), base[:40, 7:90].t(),
                 base[:1].expand(9, 300), base[:, ::2], base[:, :1].expand(70, 40)):
        check_quantized(mx.quantize(view), host(view))
        check_quantized(mx.quantize(view, along=0), host(view).T)
    x3 = tensor((3, 5, 64), t)
    check_quantized(mx.quantize(x3), host(x3).reshape(15, 64))
    check_quantized(mx.quantize(x3.transpose(0, 1)), host(x3.transpose(0, 1)).reshape(15, 64))
    flat = torch.empty(70 * 300 + 1, dtype=t, device="cuda")[1:].view(70, 300).copy_(base)  # off a 16-byte boundary
    check_quantized(mx.quantize(flat), host(flat))
    check_quantized(mx.quantize_both(flat)[1], host(flat).T)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_dequantize(shape, name):
    t = TYPES[name]
    rng = np.random.default_rng(shape[0] * 1000 + shape[1])
    rows, cols = shape
    blocks = O.blocks_of(cols)
    for fmt, width in (("mxfp4", 16), ("mxint8", 32)):
        codes = rng.integers(0, 256, (rows, blocks * width), dtype=np.uint8)
        scale = rng.integers(100, 140, (rows, blocks), dtype=np.uint8)
        scale.flat[::7] = rng.integers(0, 256, scale.flat[::7].shape, dtype=np.uint8)
        scale.flat[::11] = 255
        scale.flat[3::13] = 0
        q = mx.MxTensor.from_rows(torch.from_numpy(codes), torch.from_numpy(scale), cols, fmt).to("cuda")
        # rounded once from 64 bits, which hold every value exactly
        want = torch.from_numpy(O.decode(codes, scale, fmt, cols))
        want = want.float().to(t) if t != torch.float32 else want.float()
        got = mx.dequantize(q, t).cpu()
        assert torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0)) and torch.equal(got.isnan(), want.isnan())
        if fmt == "mxfp4":
            got = mx.dequantize(q, t, transpose=True).cpu()
            assert torch.equal(got.nan_to_num(7.0), want.t().nan_to_num(7.0))
            assert torch.equal(got.isnan(), want.t().isnan())


def check_product(y, a, b, slack=0.0):
    """y against a b^T, given as the values that both operands stand for."""
    want = a @ b.T
    bound = a.shape[1] * 2.0 ** -23 * (np.abs(a) @ np.abs(b).T)
    half = HALF_STEP[y.dtype]
    # below the normal range a rounding is half a subnormal step, whatever the value
    floor = torch.finfo(y.dtype).smallest_normal * half
    got = host(y)
    assert got.shape == want.shape
    off = np.abs(got - want) - (bound * (1 + half) + half * np.abs(want) + floor)
    assert off.max() <= 0, f"worst excess {off.max()} at {np.unravel_index(off.argmax(), off.shape)}"


PRODUCTS = [(1, 1, 1), (1, 128, 256), (1, 130, 64), (7, 128, 32), (8, 300, 100), (9, 129, 512), (16, 256, 31),
            (17, 1000, 320), (33, 127, 1024), (64, 64, 4096), (65, 257, 200), (100, 384, 768), (128, 128, 128),
            (129, 200, 300), (300, 520, 1000), (1, 4096, 4096), (5, 11008, 96), (1000, 70, 70), (2, 3000, 8192),
            (520, 1100, 2080)]


@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_matmul(m, n, k):
    a, b = tensor((m, k), torch.float32, 1), tensor((n, k), torch.bfloat16, 2)
    qa, qb = mx.quantize(a), mx.quantize(b)
    ra, rb = O.rounded(host(a)), O.rounded(host(b))
    for t in TYPES.values():
        check_product(mx.matmul(qa, qb, dtype=t), ra, rb)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_linear(m, n, k, name):
    t = TYPES[name]
    x, w = tensor((m, k), t, 3), tensor((n, k), torch.float32, 4, std=0.02)
    qw = mx.quantize(w)
    y = mx.linear(x, qw)
    assert y.dtype == t and torch.equal(y, mx.linear(x, qw)), "the order of the sums is fixed"
    check_product(y, O.rounded(host(x)), O.rounded(host(w)))
    assert torch.equal(y, mx.matmul(mx.quantize(x), qw, dtype=t))


# pairs of SMs with 256, 192 and 128 rows a tile (one round of tiles and more,
# widths that 16-byte stores fit and do not), and single CTAs with a split
MANY_ROWS = [(1003, 4101, 520), (2000, 4104, 64), (1500, 5000, 96), (700, 8200, 130), (300, 9001, 520), (129, 129, 33),
             (520, 1100, 2080), (300, 300, 257), (180, 300, 4000), (257, 1000, 3000), (1100, 10000, 70)]


@pytest.mark.parametrize("m,n,k", MANY_ROWS)
def test_many_rows(m, n, k):
    x, w = tensor((m, k), torch.bfloat16, 50), mx.quantize(tensor((n, k), torch.float32, 51, std=0.02))
    a, b = O.rounded(host(x)), O.rounded(host(tensor((n, k), torch.float32, 51, std=0.02)))
    for t in (torch.float16, torch.float32):
        y = mx.linear(x, w, dtype=t)
        assert torch.equal(y, mx.linear(x, w, dtype=t))
        check_product(y, a, b)


def test_result_rows_do_not_depend_on_their_company():
    """Rows of a batch that a kernel takes whole (no split along K) are those of
    the same rows in a larger one."""
    x, w = tensor((512, 256), torch.bfloat16, 52), mx.quantize(tensor((384, 256), torch.float32, 53))
    y = mx.linear(x, w)
    for m in (1, 7, 16, 33, 128, 129, 300):
        assert torch.equal(mx.linear(x[:m], w), y[:m])


@pytest.mark.parametrize("m,n,k", [(1, 512, 2048), (40, 1000, 4096), (700, 8200, 512)])
def test_wait_that_runs_out_is_reported_by_the_next_product(m, n, k):
    """A withheld copy: the kernel's bounded waits run out, it leaves by itself,
    the next product reports it and the one after is right again."""
    from sym_b200 import _native, pyreloc

    x, w = tensor((m, k), torch.float16, 54), mx.quantize(tensor((n, k), torch.float32, 55))
    want = mx.linear(x, w)
    torch.cuda.synchronize()
    _native.cuda_layer().sbc_test_withhold_mx(20_000_000)
    mx.linear(x, w)
    torch.cuda.synchronize()
    with pytest.raises(pyreloc.TransferError) as e:
        mx.linear(x, w)
    assert e.value.code == "backend_failure"
    assert torch.equal(mx.linear(x, w), want)


def test_linear_leading_axes_and_result_type():
    w = mx.quantize(tensor((96, 64), torch.bfloat16, 5))
    x = tensor((2, 3, 64), torch.bfloat16, 6)
    y = mx.linear(x, w, dtype=torch.float32)
    assert y.shape == (2, 3, 96) and y.dtype == torch.float32
    assert torch.equal(y.view(6, 96), mx.linear(x.view(6, 64), w, dtype=torch.float32))
    assert torch.equal(mx.linear(x[0, 0], w), mx.linear(x[0, :1], w)[0])
    wide = tensor((7, 200), torch.bfloat16, 7)
    for view in (wide[:, 40:104], wide[:, 3:67], wide[::2, :64], wide[:1, :64].expand(5, 64), wide[:, ::2][:, :64]):
        assert torch.equal(mx.linear(view, w), mx.linear(view.contiguous(), w))


def test_no_rows_and_non_finite_rows():
    w = tensor((130, 96), torch.float32, 8)
    qw = mx.quantize(w)
    for shape in ((0, 96), (2, 0, 96)):
        y = mx.linear(torch.empty(shape, dtype=torch.float16, device="cuda"), qw)
        assert y.shape == (*shape[:-1], 130)
    assert mx.quantize(torch.empty(0, 96, device="cuda")).shape == (0, 96)
    assert mx.dequantize(mx.quantize(torch.empty(0, 96, device="cuda")), torch.float32).shape == (0, 96)
    assert mx.silu_mul(torch.empty(0, 96, device="cuda")).shape == (0, 48)
    # a row with an infinity or a NaN gives NaN in its own row only; the same for a weight row
    x = tensor((5, 96), torch.float16, 9)
    x[1, 40], x[3, 95] = float("inf"), float("nan")
    y = mx.linear(x, qw)
    assert y[[1, 3]].isnan().all() and y[[0, 2, 4]].isfinite().all()
    w[129, 0] = float("-inf")
    y = mx.linear(x[:1], mx.quantize(w))
    assert y[0, 129].isnan() and y[0, :129].isfinite().all()
    # a row of zeros, and one of the smallest numbers
    x[0], x[2] = 0, 0
    x[2, 7] = torch.finfo(torch.float16).smallest_normal * 2.0 ** -10
    check_product(mx.linear(x[[0, 2, 4]], qw), O.rounded(host(x[[0, 2, 4]])), O.rounded(host(tensor((130, 96), torch.float32, 8))))


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (5, 40, 100), (128, 128, 128), (130, 257, 96), (333, 520, 700)])
def test_training_product(m, n, k, name):
    t = TYPES[name]
    x, w = tensor((m, k), t, 10).requires_grad_(), tensor((n, k), t, 11, std=0.05).requires_grad_()
    dy = tensor((m, n), t, 12, std=0.1)
    y = mx.linear(x, w)
    y.backward(dy)
    check_product(y, O.rounded(host(x)), O.rounded(host(w)))
    check_product(x.grad, O.rounded(host(dy)), O.rounded(host(w).T))
    check_product(w.grad, O.rounded(host(dy).T), O.rounded(host(x).T))
    assert x.grad.dtype == t and w.grad.dtype == t
    # one gradient alone, the same weight twice, a weight that is not trained
    gx, = torch.autograd.grad(mx.linear(x, w.detach()), x, dy)
    gw, = torch.autograd.grad(mx.linear(x.detach(), w), w, dy)
    assert torch.equal(gx, x.grad) and torch.equal(gw, w.grad)
    twice, = torch.autograd.grad((mx.linear(x.detach(), w), mx.linear(x.detach(), w)), w, (dy, dy))
    assert torch.equal(twice, (gw.float() * 2).to(t))
    q, qt = mx.quantize_both(w)
    frozen = mx.linear(x, q, qt)
    gx, = torch.autograd.grad(frozen, x, dy)
    assert torch.equal(frozen, y) and torch.equal(gx, x.grad)


def test_training_product_broadcast_gradient_and_types():
    x, w = tensor((4, 6, 64), torch.bfloat16, 13).requires_grad_(), tensor((96, 64), torch.float32, 14).requires_grad_()
    y = mx.linear(x, w)
    assert y.dtype == torch.bfloat16
    y.sum().backward()  # a gradient with strides of 0
    assert x.grad.shape == x.shape and x.grad.dtype == torch.bfloat16 and w.grad.dtype == torch.float32
    ones = np.ones((24, 96))
    check_product(w.grad, O.rounded(ones.T), O.rounded(host(x).reshape(24, 64).T))
    check_product(x.grad.view(24, 64), O.rounded(ones), O.rounded(host(w).T))


def test_training_product_gradients_against_differences():
    """On values that mxfp4 holds exactly in both directions (largest 4 in every
    block, so the scale is 1), the product is linear: differences of the loss
    between two such points are its gradient, exactly."""
    g = torch.Generator().manual_seed(3)
    grid = torch.tensor([0.0, 0.5, 1, 1.5, 2, 3, -0.5, -1, -2, -3])

    def exact(r, c):
        v = grid[torch.randint(len(grid), (r, c), generator=g)]
        v[::32, :], v[:, ::32] = 4.0, 4.0
        return v

    x, w, dy = exact(64, 64).cuda(), exact(96, 64).cuda(), exact(64, 96).cuda()
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    mx.linear(xg, wg).backward(dy)
    loss = lambda a, b: (mx.linear(a, b).double() * dy.double()).sum().item()  # noqa: E731
    base = loss(x, w)
    for i, j in ((1, 1), (5, 40), (63, 33), (33, 63), (40, 9)):
        for m, grad in ((x, xg.grad), (w, wg.grad)):
            moved = m.clone()
            moved[i, j] = 1.0 if m[i, j] != 1.0 else 2.0
            change = loss(moved, w) - base if m is x else loss(x, moved) - base
            assert change == (moved[i, j] - m[i, j]).item() * grad[i, j].item()


def silu(g):
    return g / (1 + np.exp(-g))


GATES = [(1, 1), (1, 32), (3, 31), (2, 100), (17, 256), (13, 1003), (64, 4096), (5, 11008)]


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("shape", GATES)
def test_silu_mul(shape, name):
    t = TYPES[name]
    gate, up = tensor(shape, t, 15, 1.5), tensor(shape, t, 16)
    dh = tensor(shape, t, 17, 0.1)
    g, u = gate.clone().requires_grad_(), up.clone().requires_grad_()
    h = mx.silu_mul(g, u)
    dg, du = torch.autograd.grad(h, (g, u), dh)
    assert torch.equal(h, mx.silu_mul(gate, up))
    # 32-bit steps: exp and the division are off by at most 2 steps each, the
    # exponent's own rounding by |g| 2^-24 relative, then at most 8 operations
    # of half a step; where |g| is large enough for that to matter, exp(-g) is
    # far from 1 on one side and s = 1 or h tiny on the other. Below the normal
    # range steps are absolute: exp and the division there are each off by at
    # most a step of 2^-149, so s by 2^-148 (first version: no such term, and
    # an s that became 0 once exp(-g) overflowed, at g < -88.7; the kernel now
    # takes exp(-|g|)), which the factors of s carry into the result; the
    # product g s rounds to half such a step and carries |u| or |dh|.
    gate64, up64, dh64 = host(gate), host(up), host(dh)
    half, tiny = HALF_STEP[t], torch.finfo(t).smallest_normal * HALF_STEP[t]
    rel = (16 + np.abs(gate64)) * 2.0 ** -24

    def near(got, want, rel, extra=0.0):
        off = np.abs(host(got) - want) - (np.abs(want) * (rel + half) * (1 + half) + extra + tiny)
        assert off.max() <= 0, off.max()

    with np.errstate(over="ignore"):
        sub = 2.0 ** -147
        near(h, silu(gate64) * up64, rel, sub * (1 + np.abs(gate64)) * np.abs(up64))
        gq, uq = O.rounded(gate64, "mxint8"), O.rounded(up64, "mxint8")
        s = 1 / (1 + np.exp(-gq))
        rel = (16 + np.abs(gq)) * 2.0 ** -24
        near(du, dh64 * gq * s, rel, sub * (1 + np.abs(gq)) * np.abs(dh64))
        # 1 + g (1 - s) cancels near its zero: its terms' size counts there
        size = np.abs(dh64 * uq) * s * (1 + np.abs(gq) * (1 - s))
        near(dg, dh64 * uq * s * (1 + gq * (1 - s)), 0.0,
             size * (rel + 2.0 ** -22) + sub * (2 + np.abs(gq)) * (1 + np.abs(dh64 * uq)))


def test_silu_mul_gradients_against_differences():
    """Inputs that mxint8 holds exactly (multiples of 2^-6 with a largest
    magnitude of 1.984375 in every block): the gradients are those of the
    function itself, found here by central differences in 64 bits."""
    g = torch.Generator().manual_seed(5)
    v = torch.randint(-127, 128, (2, 6, 64), generator=g).double() / 64
    v[..., ::32] = 127 / 64
    gate, up = v[0].float().cuda().requires_grad_(), v[1].float().cuda().requires_grad_()
    dg, du = torch.autograd.grad(mx.silu_mul(gate, up).sum(), (gate, up))
    a, b, d = v[0].numpy(), v[1].numpy(), 1e-5
    want_g = (silu(a + d) - silu(a - d)) / (2 * d) * b
    # the differences' own error: d^2 |f'''| / 6 < 1e-10 and rounding 1e-16 / d; the kernel's: 32-bit steps
    assert np.abs(host(dg) - want_g).max() < 1e-9 + 2.0 ** -19
    assert np.abs(host(du) - silu(a)).max() < 2.0 ** -19


@pytest.mark.parametrize("name", TYPES)
def test_silu_mul_halves_of_one_tensor_and_strides(name):
    t = TYPES[name]
    both = tensor((3, 5, 2 * 72), t, 18)
    p = both.clone().requires_grad_()
    g, u = (x.clone().requires_grad_() for x in both.chunk(2, -1))
    dh = tensor((3, 5, 72), t, 19)
    h = mx.silu_mul(p)
    dp, = torch.autograd.grad(h, p, dh)
    dg, du = torch.autograd.grad(mx.silu_mul(g, u), (g, u), dh)
    assert torch.equal(h, mx.silu_mul(*both.chunk(2, -1)))
    assert torch.equal(dp, torch.cat((dg, du), -1))
    dp2, = torch.autograd.grad(mx.silu_mul(p), p, dh[:1, :1, :1].expand(3, 5, 72))
    dp3, = torch.autograd.grad(mx.silu_mul(p), p, dh[:1, :1, :1].expand(3, 5, 72).contiguous())
    assert torch.equal(dp2, dp3)
    odd = tensor((9, 101), t, 20)
    assert torch.equal(mx.silu_mul(odd[:, 1:41], odd[:, 50:90]), mx.silu_mul(odd[:, 1:41].clone(), odd[:, 50:90].clone()))
    same, = torch.autograd.grad(mx.silu_mul(p, p), p, torch.ones_like(p))  # one tensor as both
    a, b = (both.clone().requires_grad_() for _ in range(2))
    da, db = torch.autograd.grad(mx.silu_mul(a, b), (a, b), torch.ones_like(a))
    assert torch.equal(same, da + db)


def test_silu_mul_infinities_stay_in_their_block():
    gate, up = tensor((2, 96), torch.float32, 21), tensor((2, 96), torch.float32, 22)
    gate[0, 3], up[1, 95] = float("inf"), float("nan")
    gate[1, 5], gate[0, 70] = -300.0, 300.0
    g, u = gate.clone().requires_grad_(), up.clone().requires_grad_()
    dg, du = torch.autograd.grad(mx.silu_mul(g, u).sum(), (g, u))
    assert dg[0, :32].isnan().all() and du[0, :32].isnan().all()
    assert dg[0, 32:].isfinite().all() and du[0, 32:].isfinite().all()
    assert dg[1, 64:].isnan().all() and dg[1, :64].isfinite().all() and du[1].isfinite().all()


def mlp(x, gate_up, down):
    return mx.linear(mx.silu_mul(mx.linear(x, gate_up)), down)


def test_feed_forward_together():
    """Products and gate as a layer uses them: training with float weights,
    then the same weights served in 4 bits with the same result."""
    x = tensor((2, 37, 128), torch.bfloat16, 23).requires_grad_()
    gate_up = tensor((2 * 352, 128), torch.bfloat16, 24, 0.1).requires_grad_()
    down = tensor((128, 352), torch.bfloat16, 25, 0.1).requires_grad_()
    y = mlp(x, gate_up, down)
    dy = tensor(y.shape, torch.bfloat16, 26)
    y.backward(dy)
    q_gate_up, q_down = mx.quantize(gate_up), mx.quantize(down)
    with torch.no_grad():
        served = mlp(x, q_gate_up, q_down)
    assert torch.equal(served, y.detach())
    # the layer by hand, from the operators' values in 64 bits; intermediate results in bf16
    a = host(mx.linear(x.detach(), q_gate_up)).reshape(74, -1)
    h = host(mx.silu_mul(mx.linear(x.detach(), q_gate_up))).reshape(74, -1)
    dyh = host(dy).reshape(74, -1)
    check_product(down.grad, O.rounded(dyh.T), O.rounded(h.T))
    dh = mx.matmul(mx.quantize(dy), mx.quantize(down, along=0), dtype=torch.bfloat16)
    gq, uq = O.rounded(a[:, :352], "mxint8"), O.rounded(a[:, 352:], "mxint8")
    with np.errstate(over="ignore"):
        s = 1 / (1 + np.exp(-gq))
    da = torch.from_numpy(np.concatenate((host(dh) * uq * s * (1 + gq * (1 - s)), host(dh) * gq * s), 1)).to(torch.bfloat16)
    got, = torch.autograd.grad(mx.silu_mul(t := torch.from_numpy(a).to(torch.bfloat16).cuda().requires_grad_()), t, dh)
    step = 2.0 ** -7  # the two may round to neighbouring values
    assert (host(got) - host(da) <= step * np.abs(host(da)) + 1e-30).all()
    check_product(gate_up.grad, O.rounded(host(got).T), O.rounded(host(x).reshape(74, -1).T))
    check_product(x.grad.view(74, -1), O.rounded(host(got)), O.rounded(host(gate_up).T))


def test_other_stream_and_two_at_once():
    x, w = tensor((9, 2048), torch.float16, 27), mx.quantize(tensor((3000, 2048), torch.float32, 28))
    want = mx.linear(x, w)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(mx.linear(x, w))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for y in got)


def test_captured_and_replayed():
    """Two graphs over the same static inputs, replayed in turn with new values
    and compared with eager steps between the replays."""
    x = tensor((33, 512), torch.bfloat16, 29).requires_grad_()
    w = tensor((256, 512), torch.bfloat16, 30, 0.05).requires_grad_()
    qw = mx.quantize(w)
    dy = tensor((33, 256), torch.bfloat16, 31)

    def serve():
        with torch.no_grad():
            return mx.silu_mul(mx.linear(x, qw))

    def step():
        y = mx.linear(x, w)
        return (y, *torch.autograd.grad(y, (x, w), dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        serve()
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for fn in (serve, step):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = fn()
        graphs.append((g, out, fn))
    for seed in (40, 41):
        with torch.no_grad():
            x.copy_(tensor((33, 512), torch.bfloat16, seed))
            dy.copy_(tensor((33, 256), torch.bfloat16, seed + 1))
        for g, _, _ in graphs:
            g.replay()
        for _, out, fn in graphs:
            want = fn()
            for a, b in zip(out if isinstance(out, tuple) else (out,), want if isinstance(want, tuple) else (want,)):
                assert torch.equal(a, b)


def test_gpu_refusals_leave_the_device_usable():
    x, w = tensor((4, 64), torch.float16), tensor((80, 64), torch.float16, 1)
    q, qt = mx.quantize_both(w)
    k8 = mx.quantize(w, "mxint8")
    xg = x.clone().requires_grad_()
    for call in (lambda: mx.linear(x[:, :32], q), lambda: mx.linear(x, k8), lambda: mx.matmul(q, k8),
                 lambda: mx.matmul(q, qt), lambda: mx.linear(xg, q), lambda: mx.linear(xg, q, q),
                 lambda: mx.linear(x, w, qt), lambda: mx.linear(x, w[0]), lambda: mx.dequantize(k8, transpose=True),
                 lambda: mx.quantize(x, "mxint8", along=0), lambda: mx.quantize(x, along=1),
                 lambda: mx.quantize(x[0], along=0), lambda: mx.quantize(x, "fp4"), lambda: mx.quantize_both(x[:0]),
                 lambda: mx.silu_mul(x, w), lambda: mx.silu_mul(x, x.float()), lambda: mx.silu_mul(x[:, :63]),
                 lambda: mx.linear(x[:, :0], q), lambda: mx.linear(x, w.cpu()),
                 lambda: mx.MxTensor(q.codes.view(-1)[1:-31].view(-1, 32), q.scales, (79, 64))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        mx.linear(x, q, dtype=torch.float64)
    assert mx.linear(x, q).isfinite().all()


def test_two_graphs_of_one_memory_pool():
    """Graphs that share a pool, and so each other's freed workspaces, replayed
    in turn."""
    xs = [tensor((m, 1024), torch.bfloat16, 60 + m) for m in (40, 200)]
    w = mx.quantize(tensor((640, 1024), torch.float32, 61, 0.05))
    want = [mx.silu_mul(mx.linear(x, w)) for x in xs]
    pool = torch.cuda.graph_pool_handle()
    graphs = []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=pool):
            out = mx.silu_mul(mx.linear(x, w))
        graphs.append((g, out))
    for turn in (0, 1, 1, 0):
        graphs[turn][0].replay()
        torch.cuda.synchronize()
        assert torch.equal(graphs[turn][1], want[turn])


def test_first_call_of_a_process_may_be_captured():
    import subprocess
    import sys
    from pathlib import Path

    code = """
import torch
from sym_b200 import microscale as mx
x = torch.ones(20, 64, device="cuda", dtype=torch.bfloat16)
codes = torch.full((96, 32), 0x22, dtype=torch.uint8, device="cuda")  # ones
w = mx.MxTensor(codes, torch.full((512,), 127, dtype=torch.uint8, device="cuda"), (96, 64))
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    y = mx.linear(x, w)
    z = mx.linear(x[:1], w)
    q, qt = mx.quantize_both(x)
g.replay()
torch.cuda.synchronize()
assert (y == 64).all() and (z == 64).all() and (mx.dequantize(qt) == 1).all()
"""
    root = Path(__file__).resolve().parent.parent
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


def test_second_derivatives_are_refused():
    x, w = tensor((8, 64), torch.float32, 62).requires_grad_(), tensor((32, 64), torch.float32, 63).requires_grad_()
    for y in (mx.linear(x, w), mx.silu_mul(x, x * 2)):
        g, = torch.autograd.grad(y.sum(), x, create_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(g.sum(), x)


def test_training_product_of_one_row_and_of_a_transposed_weight():
    x, w = tensor((64,), torch.float16, 64).requires_grad_(), tensor((64, 40), torch.float16, 65).requires_grad_()
    y = mx.linear(x, w.t())
    dy = tensor((40,), torch.float16, 66)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    assert y.shape == (40,) and dx.shape == (64,) and dw.shape == (64, 40)
    row, wt = host(x)[None], host(w).T
    check_product(y[None], O.rounded(row), O.rounded(wt))
    check_product(dx[None], O.rounded(host(dy)[None]), O.rounded(wt.T))
    check_product(dw.t(), O.rounded(host(dy)[None].T), O.rounded(row.T))


def test_large_offsets():
    """Codes, values and results beyond 2^31 elements: the last rows agree with
    the same rows alone."""
    rows, cols = 70_000, 32_768
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda")
    x[:-3].fill_(1.0)
    x[-3:] = tensor((3, cols), torch.bfloat16, 67)
    q, qt = mx.quantize_both(x)
    alone = mx.quantize(x[-3:])
    assert torch.equal(q.codes[-3:], alone.codes)
    last = mx.dequantize(q, torch.bfloat16)[-3:]
    assert torch.equal(last, mx.dequantize(alone, torch.bfloat16))
    del q
    # the transposed form: the last block of every column holds the last rows
    tail = mx.quantize(x[-(rows % 32 or 32):], along=0)
    assert torch.equal(qt.codes[:, -16:], tail.codes)
    wide = mx.dequantize(qt, torch.bfloat16, transpose=True)
    assert torch.equal(wide[-3:], mx.dequantize(tail, torch.bfloat16, transpose=True)[-3:])
    del wide, qt
    h = mx.silu_mul(x, x)
    assert torch.equal(h[-3:], mx.silu_mul(x[-3:], x[-3:]))
    del h
    w = mx.quantize(tensor((64, cols), torch.bfloat16, 68, 0.05))
    y = mx.linear(x, w)
    assert torch.equal(mx.linear(x[-300:], w)[-3:], mx.linear(x[-300:].clone(), w)[-3:])
    a, b = O.rounded(host(x[-3:])), O.rounded(host(tensor((64, cols), torch.bfloat16, 68, 0.05)))
    check_product(y[-3:], a, b)


def test_training_product_without_rows():
    """A batch of no rows (an expert that got no tokens): empty result, zero
    weight gradient."""
    w = tensor((40, 64), torch.bfloat16, 70).requires_grad_()
    for shape in ((0, 64), (2, 0, 64)):
        x = torch.empty(shape, dtype=torch.bfloat16, device="cuda", requires_grad=True)
        y = mx.linear(x, w)
        dx, dw = torch.autograd.grad(y, (x, w), torch.empty_like(y))
        assert y.shape == (*shape[:-1], 40) and dx.shape == shape and torch.equal(dw, torch.zeros_like(w))
        q, qt = mx.quantize_both(w)
        assert torch.autograd.grad(mx.linear(x, q, qt).sum(), x)[0].shape == shape
    g = torch.empty(0, 64, device="cuda", requires_grad=True)
    assert torch.autograd.grad(mx.silu_mul(g, g).sum(), g)[0].shape == (0, 64)


def test_copies_of_a_matrix_own_their_memory():
    import copy
    import pickle

    x = tensor((5, 256), torch.float16, 71)
    q = mx.quantize(tensor((300, 256), torch.float32, 72))
    want = mx.linear(x, q)
    copies = [copy.deepcopy(q), pickle.loads(pickle.dumps(q)), q.to("cpu").to("cuda"), copy.copy(q)]
    for c in copies[:3]:
        assert c.codes.data_ptr() != q.codes.data_ptr()
        c_native = c.native
        assert c_native.codes == c.codes.data_ptr() and c_native.scales == c.scales.data_ptr()
    for name in ("codes", "scales", "shape", "format", "native"):
        with pytest.raises(AttributeError):
            setattr(q, name, None)
    del q
    torch.cuda.empty_cache()
    for c in copies:
        assert torch.equal(mx.linear(x, c), want)


@pytest.mark.parametrize("rows,cols", [(128, 40), (40, 128), (256, 129), (128, 1)])
def test_absent_blocks_have_scale_zero(rows, cols):
    """The bytes of a row's last scale tile that belong to no block are 0, in
    either direction: a product may read them beside zero codes."""
    x = tensor((rows, cols), torch.bfloat16, 73).abs() + 1  # no block has the scale byte 0
    for q in (mx.quantize(x), mx.quantize(x, along=0), *mx.quantize_both(x)):
        r, c = q.shape
        blocks, quads = O.blocks_of(c), -(-c // 128)
        tiles = q.scales.view(-(-r // 128), quads, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(-1, quads * 4)[:r]
        assert (tiles[:, :blocks] > 0).all() and (tiles[:, blocks:] == 0).all()
