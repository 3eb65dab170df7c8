"""A feed-forward layer's steps at once from several threads on streams of their
own, and captured whole: the results of the same steps one by one."""
import threading

import pytest
import torch

from sym_b200 import microscale as mx

pytestmark = pytest.mark.gpu


class Layer:
    """rows x 160 -> 2 x 352 gated -> 160; weights frozen in 4 bits or trained."""

    def __init__(self, rows, seed):
        g = torch.Generator().manual_seed(seed)
        draw = lambda *s, std=1.0: (torch.randn(*s, generator=g) * std).bfloat16().cuda()  # noqa: E731
        self.x = draw(rows, 160).requires_grad_()
        self.gate_up, self.down = draw(704, 160, std=0.1).requires_grad_(), draw(160, 352, std=0.1).requires_grad_()
        self.dy = draw(rows, 160)
        self.frozen = [mx.quantize_both(w) for w in (self.gate_up, self.down)]

    def trained(self):
        y = mx.linear(mx.silu_mul(mx.linear(self.x, self.gate_up)), self.down)
        return (y.detach(), *torch.autograd.grad(y, (self.x, self.gate_up, self.down), self.dy))

    def adapted(self):
        y = mx.linear(mx.silu_mul(mx.linear(self.x, *self.frozen[0])), *self.frozen[1])
        return y.detach(), torch.autograd.grad(y, self.x, self.dy)[0]

    def served(self):
        with torch.no_grad():
            return (mx.linear(mx.silu_mul(mx.linear(self.x, self.frozen[0][0])), self.frozen[1][0]),
                    mx.linear(mx.silu_mul(mx.linear(self.x, self.gate_up)), self.down))

    def steps(self):
        return [t for step in (self.trained, self.adapted, self.served) for t in step()]


ROWS = (1, 5, 33, 130, 700)


def test_steps_at_once_from_threads_on_their_own_streams():
    layers = [Layer(m, i) for i, m in enumerate(ROWS)]
    want = [layer.steps() for layer in layers]
    torch.cuda.synchronize()
    wrong = []

    def work(layer, want):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(12):
                    got = layer.steps()
                    torch.cuda.current_stream().synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, want)):
                        wrong.append(layer.x.shape[0])
        except Exception as e:  # noqa: BLE001
            wrong.append(e)

    threads = [threading.Thread(target=work, args=a) for a in zip(layers, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    mx.check()
    assert not wrong, wrong


@pytest.mark.parametrize("rows", ROWS)
def test_whole_steps_captured_and_replayed(rows):
    layer = Layer(rows, 7)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer.steps()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = layer.steps()
    for seed in (8, 9):
        other = Layer(rows, seed)
        with torch.no_grad():
            layer.x.copy_(other.x)
            layer.dy.copy_(other.dy)
            layer.down.copy_(other.down)
        for _ in range(3):
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, layer.steps()))
    mx.check()
