"""Calls of the training operators that the documentation allows beside the ordinary ones, as far as the host decides
them.  No GPU."""

import threading

import torch

from backendbench_amd.ops import _common, elementwise


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


def test_out_tensors_with_memory_in_common_are_seen():
    base = torch.zeros(6, 8)
    meets = elementwise._meet
    assert meets([base, base]) and meets([base[:3], base[2:]]) and meets([base[1], torch.zeros(2), base[1, 4:]])
    assert meets([base[:, :2], base[:, 2:]])  # interleaved: a span, not an element list
    assert not meets([base[:3], base[3:]]) and not meets([base[0], base[5], torch.zeros(8)]) and not meets([base[:0], base])
