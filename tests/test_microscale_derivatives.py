"""Microscaled calls under torch's other derivatives and its recorders: what
cannot be right is refused, what is recorded gives the call's result.

The CPU tests need no CUDA tensor: such a call is refused before its tensors
are looked at, where it used to go on to the tensors' addresses."""
import pytest
import torch
import torch.autograd.forward_ad as fw
from torch.fx.experimental.proxy_tensor import make_fx

from sym_b200 import microscale as mx


def host_matrix(rows=4, cols=64):
    return mx.MxTensor(torch.zeros(rows, cols // 2, dtype=torch.uint8), torch.zeros(512, dtype=torch.uint8), (rows, cols))


def test_forward_mode_tangents_are_refused():
    x, w, q = torch.ones(2, 64), torch.ones(4, 64), host_matrix()
    with fw.dual_level():
        d = fw.make_dual(x, torch.ones_like(x))
        for call in (lambda: mx.linear(d, q), lambda: mx.linear(d, q, q), lambda: mx.linear(d, w),
                     lambda: mx.linear(x, fw.make_dual(w, w)), lambda: mx.silu_mul(d), lambda: mx.silu_mul(x, d)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        with pytest.raises(ValueError, match="CUDA"):
            mx.linear(x, q)  # without a tangent it is an ordinary call


@pytest.mark.parametrize("pre_dispatch", (False, True))
def test_make_fx_is_refused(pre_dispatch):
    x, q = torch.ones(2, 64), host_matrix()
    for call in (lambda x: mx.linear(x, q), lambda x: mx.linear(x, x), lambda x: mx.silu_mul(x),
                 lambda x: mx.quantize(x).codes, lambda x: mx.quantize_both(x)[0].codes, lambda x: mx.dequantize(q),
                 lambda x: mx.matmul(q, q)):
        with pytest.raises(NotImplementedError, match="make_fx"):
            make_fx(call, pre_dispatch=pre_dispatch)(x)


def test_tracing_of_calls_that_are_no_autograd_functions_is_refused():
    x, q = torch.ones(2, 64), host_matrix()
    for call in (lambda x: mx.quantize(x).codes, lambda x: mx.quantize_both(x)[0].codes, lambda x: mx.dequantize(q),
                 lambda x: mx.matmul(q, q)):
        with pytest.raises(NotImplementedError, match="jit"):
            torch.jit.trace(call, (x,), check_trace=False)


def test_make_fx_of_a_backward_pass_is_refused():
    """Also where the forward pass was not recorded."""
    dy = torch.ones(2, 64)
    for function in (mx._FrozenLinear, mx._TrainLinear, mx._SiluMul):
        for pre_dispatch in (False, True):
            with pytest.raises(NotImplementedError, match="make_fx"):
                make_fx(lambda dy: function.backward(None, dy), pre_dispatch=pre_dispatch)(dy)


def test_tangents_of_incoming_gradients_are_refused():
    dy = torch.ones(2, 64)
    with fw.dual_level():
        dual = fw.make_dual(dy, dy)
        for function in (mx._FrozenLinear, mx._TrainLinear, mx._SiluMul):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                function.backward(None, dual)


def test_other_dispatch_modes_are_no_recorders():
    from torch.utils.flop_counter import FlopCounterMode

    with FlopCounterMode(display=False), pytest.raises(ValueError, match="CUDA"):
        mx.silu_mul(torch.ones(2, 64))


def tensor(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).cuda()


@pytest.mark.gpu
def test_traces_give_the_calls_results():
    x, w = tensor(5, 64), tensor(96, 64, seed=1)
    q, qt = mx.quantize_both(w)
    other = tensor(5, 64, seed=2)
    for call in (lambda x: mx.linear(x, q) + 1, lambda x: mx.linear(x, q, qt) + 1, lambda x: mx.silu_mul(x) * 2,
                 lambda x: mx.silu_mul(x, x + 1), lambda x: mx.linear(x, w), lambda x: mx.silu_mul(mx.linear(x, q))):
        traced = torch.jit.trace(call, (x,), check_trace=False)
        for _ in range(3):  # the first runs of a trace are its profiling ones
            torch.empty(1 << 20, device="cuda").fill_(float("nan"))  # what an allocation alone would hold
            assert torch.equal(traced(other), call(other))
    xg = x.clone().requires_grad_()
    traced = torch.jit.trace(lambda x: mx.linear(x, q, qt), (xg,), check_trace=False)
    dy = tensor(5, 96, seed=3)
    want, = torch.autograd.grad(mx.linear(xg, q, qt), xg, dy)
    got, = torch.autograd.grad(traced(xg), xg, dy)
    assert torch.equal(got, want)
    without = torch.jit.trace(lambda x: mx.linear(x, q), (x,), check_trace=False)
    with pytest.raises(Exception, match="weight_t"):
        torch.autograd.grad(without(xg).sum(), xg)


@pytest.mark.gpu
def test_forward_mode_and_transforms_on_the_gpu():
    x, w = tensor(5, 64), tensor(96, 64, seed=1)
    q = mx.quantize(w)
    with fw.dual_level():
        d = fw.make_dual(x, torch.ones_like(x))
        for call in (lambda: mx.linear(d, q), lambda: mx.linear(d, w), lambda: mx.silu_mul(d)):
            with pytest.raises(NotImplementedError):
                call()
        assert torch.equal(mx.linear(x, q), mx.linear(fw.unpack_dual(d).primal, q))
    for call in (lambda x: mx.linear(x, q), lambda x: mx.silu_mul(x), lambda x: mx.linear(x, w)):
        with pytest.raises((RuntimeError, NotImplementedError)):
            torch.func.jvp(call, (x,), (x,))
        with pytest.raises(RuntimeError):
            torch.func.vmap(call)(x.view(5, 1, 64))
        for mode in ("real", "fake", "symbolic"):
            with pytest.raises((RuntimeError, NotImplementedError)):
                make_fx(call, tracing_mode=mode)(x)


@pytest.mark.gpu
def test_recorded_backward_passes_on_the_gpu():
    x, w = tensor(5, 64).requires_grad_(), tensor(96, 64, seed=1)
    q, qt = mx.quantize_both(w)
    for y in (mx.linear(x, q, qt), mx.linear(x, w), mx.silu_mul(x)):
        dy = torch.ones_like(y)
        with pytest.raises(NotImplementedError):
            make_fx(lambda dy: torch.autograd.grad(y, x, dy, retain_graph=True)[0])(dy)
        with fw.dual_level():
            with pytest.raises(NotImplementedError):
                torch.autograd.grad(y, x, fw.make_dual(dy, dy), retain_graph=True)
        assert torch.autograd.grad(y, x, dy)[0].isfinite().all()


@pytest.mark.gpu
def test_compiled_regions_run_the_calls_between_their_graphs():
    x, w = tensor(5, 64), tensor(96, 64, seed=1)
    q, qt = mx.quantize_both(w)

    def layer(x, w):
        a = mx.linear(x * 2, w) + 1
        b = mx.linear(torch.sin(x), q, qt)
        return mx.silu_mul(a, b).sum()

    xs = [x.clone().requires_grad_() for _ in range(2)]
    ws = [w.clone().requires_grad_() for _ in range(2)]
    compiled = torch.compile(layer, backend="eager")
    for _ in range(2):
        want = torch.autograd.grad(layer(xs[0], ws[0]), (xs[0], ws[0]))
        got = torch.autograd.grad(compiled(xs[1], ws[1]), (xs[1], ws[1]))
        assert torch.equal(compiled(xs[1], ws[1]), layer(xs[0], ws[0]))
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    with torch.no_grad():
        for call in (lambda x: mx.linear(x, q) * 2, lambda x: mx.quantize(x).codes.clone(),
                     lambda x: mx.quantize_both(x + 1)[1].codes + 1,
                     lambda x: mx.dequantize(mx.quantize(x * 2), torch.float32) + 1,
                     lambda x: mx.matmul(mx.quantize(x, along=0), mx.quantize(x + 1, along=0)) * 2,
                     lambda x: mx.linear(x, mx.MxTensor(q.codes.clone(), q.scales.clone(), (96, 64))) + 1,
                     lambda x: mx.linear(x, mx.MxTensor.from_rows(q.codes.clone(), q.row_scales(), 64)) + 1,
                     lambda x: mx.linear(x, q.to("cpu").to("cuda")) + 1):
            assert torch.equal(torch.compile(call, backend="eager")(x), call(x))
            torch._dynamo.reset()
