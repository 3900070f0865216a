"""Calls of the training operators that the documentation allows beside the ordinary ones, on the GPU, against the float64
definitions with the tolerances of tests/test_training_gpu.py."""

import threading

import pytest
import torch

from backendbench_amd import ops
from backendbench_amd.ops import elementwise
from test_training_gpu import generator, ln_case, ln_check, randn

pytestmark = pytest.mark.gpu


def test_layer_norm_backward_beside_an_out_overload_on_another_thread():
    """While one thread is inside an out= overload, gradients of the same shapes on another go into tensors of their own."""
    rows, cols = 37, 768
    dy, x, mean, rstd, w, b = ln_case(rows, cols, torch.float32, torch.float32, 51)
    inside, done, box = threading.Event(), threading.Event(), []

    def slow(t):
        inside.set()
        assert done.wait(60)
        return t + 1.0

    outs = [torch.full_like(t, 3.0) for t in (x, w)]
    worker = [threading.Thread(target=lambda o=o: box.append(elementwise.out_variant(slow)(torch.zeros_like(o), out=o))) for o in outs]
    try:
        for t in worker:
            t.start()
        assert inside.wait(60)
        got = ops.native_layer_norm_backward(dy, x, [cols], mean, rstd, w, b, [True] * 3)
    finally:
        done.set()
        for t in worker:
            t.join()
    ln_check(got, dy, x, mean, rstd, w, rows, cols, "beside an out= overload")
    assert len(box) == 2 and all((o == 1.0).all() for o in outs)
    assert not {t.data_ptr() for t in got} & {o.data_ptr() for o in outs}


def test_layer_norm_backward_into_out_tensors_that_share_memory():
    """Results that go to the same memory are stored one after the other: the last one stands, whole."""
    rows, cols = 300, 512
    dy, x, mean, rstd, w, b = ln_case(rows, cols, torch.float32, torch.float32, 52)
    same, dx = torch.full_like(w, 3.0), torch.full_like(x, 3.0)
    ops.native_layer_norm_backward_out(dy, x, [cols], mean, rstd, w, b, [True] * 3, out0=dx, out1=same, out2=same)
    ln_check([dx, None, same], dy, x, mean, rstd, w, rows, cols, "one tensor twice")
    part = torch.full((cols + 64,), 3.0, device="cuda")
    ops.native_layer_norm_backward_out(dy, x, [cols], mean, rstd, w, b, [True] * 3, out0=dx, out1=part[:cols], out2=part[64:])
    ln_check([dx, None, part[64:]], dy, x, mean, rstd, w, rows, cols, "overlapping")
