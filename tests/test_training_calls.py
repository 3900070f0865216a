"""Calls of the training operators that the documentation allows beside the ordinary ones, as far as the host decides
them.  No GPU."""

import threading

import pytest
import torch

from backendbench_amd import _lib
from backendbench_amd.ops import _common, elementwise, training
from oracle import training_ref as ref


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


ONE_ROW = {
    "a column's transpose": lambda k: torch.randn(k, 1).t(),
    "the first of a row repeated": lambda k: torch.randn(k).expand(4, k)[:1],
    "a far odd row": lambda k: torch.randn(3, k + 5)[1:2, :k],
    "overlapping": lambda k: torch.randn(k).as_strided((1, k), (0, 1)),
}


@pytest.mark.parametrize("what", ONE_ROW)
@pytest.mark.parametrize("k", [1, 7, 16])
def test_one_row_has_no_distance(what, k):
    """A row's distance to the next means nothing where there is one row, whatever stride torch reports."""
    t = ONE_ROW[what](k)
    rows = training._rows_of(t)
    assert rows.shape == (1, k) and rows.stride() == (k, 1) and rows.data_ptr() == t.data_ptr() and torch.equal(rows, t)


def test_c_entry_points_take_one_row_of_any_stride():
    """Past the check of overlapping rows: refused for its type (forward) or its workspace (backward), nothing launched."""
    lib, p = _lib.load(), 1 << 20
    for stride in (0, 1, 63):
        assert lib.mi355_gated_linear(p, stride, p, 64, p, None, 1, 8, 64, 0, _lib.I8, None) == -2
        assert lib.mi355_gated_linear(p, stride, p, 64, p, None, 2, 8, 64, 0, _lib.I8, None) == -1
        for rows, text in ((1, b"workspace"), (2, b"overlap")):
            assert lib.mi355_gated_linear_backward(p, p, stride, p, 64, p, p, p, rows, 8, 64, 0, _lib.F32, p, 0, None) == -1
            assert text in lib.mi355_last_error()


@pytest.mark.parametrize("halves,t", [(1, 0), (3, 2), (5, 2), (7, 4), (131071, 65536)])
def test_dropout_probabilities_halfway_between_two_steps(halves, t):
    """p in the middle of two 65536ths goes to the even one, as the definition's round() does."""
    p = halves * 2.0 ** -17
    assert ref.dropout_scale(p) == (65536.0 / (65536 - t) if t < 65536 else 0.0)
    n = 1 << 12
    dropped = n - int(ref.dropout_keep(n, p, 3, 0).sum())
    assert dropped == (0 if t == 0 else n) or 0 < t < 65536
