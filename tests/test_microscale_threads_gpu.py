"""Microscaled calls as the first CUDA work of a thread: a worker's first
token, and the backward pass, which torch runs in a thread of its own."""
import subprocess
import sys
import threading
from pathlib import Path

import pytest
import torch

from sym_b200 import microscale as mx

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parent.parent


def in_new_thread(call):
    out = []

    def run():
        try:
            out.append(call())
        except Exception as e:  # noqa: BLE001
            out.append(e)

    t = threading.Thread(target=run)
    t.start()
    t.join()
    return out[0]


@pytest.mark.parametrize("rows", (1, 5, 40, 300))
def test_first_call_of_a_thread(rows):
    g = torch.Generator().manual_seed(rows)
    x = torch.randn(rows, 64, generator=g).cuda()
    w = torch.randn(96, 64, generator=g).cuda()
    q, qx = mx.quantize(w), mx.quantize(x)
    y = mx.linear(x, q)
    torch.cuda.synchronize()
    for call, want in ((lambda: mx.linear(x, q), y), (lambda: mx.matmul(qx, q, dtype=x.dtype), y),
                       (lambda: mx.quantize(x).codes, qx.codes), (lambda: mx.dequantize(q), mx.dequantize(q)),
                       (lambda: mx.silu_mul(x), mx.silu_mul(x))):
        got = in_new_thread(call)
        torch.cuda.synchronize()
        assert isinstance(got, torch.Tensor), got
        assert torch.equal(got, want)


@pytest.mark.parametrize("rows", (1, 5, 40))
def test_first_backward_pass_of_a_process(rows):
    code = f"""
import torch
from sym_b200 import microscale as mx
w = torch.randn(96, 64, generator=torch.Generator().manual_seed(0)).cuda()
x = torch.randn({rows}, 64, generator=torch.Generator().manual_seed(1)).cuda().requires_grad_()
dy = torch.randn({rows}, 96, generator=torch.Generator().manual_seed(2)).cuda()
q, qt = mx.quantize_both(w)
y = mx.linear(x, q, qt)
got, = torch.autograd.grad(y, x, dy)
assert torch.equal(got, mx.linear(dy, qt))
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
