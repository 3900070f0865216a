"""Calls of the training operators that the documentation allows beside the ordinary ones, as far as the host decides
them.  No GPU."""

import threading

import torch

from backendbench_amd.ops import _common


def on_another_thread(fn):
    box = []
    t = threading.Thread(target=lambda: box.append(fn()))
    t.start()
    t.join()
    return box[0]


def test_an_offered_out_tensor_is_its_threads_own():
    """A result buffer asked for on one thread (autograd's workers run gradients) is never the out tensor of another's call."""
    out, cpu = torch.zeros(3, 4), torch.device("cpu")
    _common.offer_out(out)
    try:
        assert on_another_thread(lambda: _common.new_result((3, 4), torch.float32, cpu)) is not out
        assert on_another_thread(lambda: _common.result_like(torch.empty(3, 4), torch.float32)) is not out
        on_another_thread(_common.withdraw_out)
        on_another_thread(lambda: _common.offer_out(torch.ones(3, 4)))
        assert _common.new_result((3, 4), torch.float32, cpu) is out
        assert _common.new_result((3, 4), torch.float32, cpu) is not out  # taken
    finally:
        _common.withdraw_out()
