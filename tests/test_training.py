"""The training operators on the host: header against binding, slots, refusals, and the oracle's formulas against
published values and against differences.  No GPU."""

import os
import re

import pytest
import torch

from backendbench_amd import _lib, ops
from backendbench_amd.backends import DirectoryBackend
from oracle import training_ref as ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def declared():
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "mi355_train.h")).read(), flags=re.S)
    return sorted(set(re.findall(r"\b(mi355_[a-z_0-9]+)\s*\(", text)))


def test_every_declared_symbol_is_exported_and_bound():
    lib = _lib.load()
    assert sorted(_lib.TRAIN_SIGNATURES) == declared()
    assert all(hasattr(lib, fn) for fn in declared())
    assert not set(_lib.TRAIN_SIGNATURES) & set(_lib.SIGNATURES)


@pytest.mark.parametrize("name,value", [("MI355_SILU", _lib.SILU), ("MI355_GELU", _lib.GELU), ("MI355_GELU_TANH", _lib.GELU_TANH)])
def test_enum_values_match_header(name, value):
    text = open(os.path.join(ROOT, "include", "mi355_train.h")).read()
    assert int(re.search(r"\b%s\s*=\s*(\d+)" % name, text).group(1)) == value


def test_training_folder_tree():
    base = os.path.join(ROOT, "generated_training_kernels")
    assert sorted(os.listdir(base)) == sorted(ops.TRAINING_SLOTS)
    b = DirectoryBackend(base)
    assert set(b.compiled_kernels) == {torch.ops.aten.native_layer_norm_backward.default, torch.ops.aten.native_layer_norm_backward.out}
    assert not set(ops.TRAINING_SLOTS) & set(ops.SLOTS)


# ---- refusals --------------------------------------------------------------------------
def ln_args(**kw):
    a = dict(grad_out=torch.zeros(3, 8), input=torch.zeros(3, 8), normalized_shape=[8], mean=torch.zeros(3, 1), rstd=torch.ones(3, 1),
             weight=torch.ones(8), bias=torch.zeros(8), output_mask=[True] * 3)
    a.update(kw)
    return a


@pytest.mark.parametrize("change,error,match", [
    (dict(normalized_shape=[7]), RuntimeError, "normalized_shape"),
    (dict(normalized_shape=[]), RuntimeError, "normalized_shape"),
    (dict(grad_out=torch.zeros(3, 7)), RuntimeError, "grad_out"),
    (dict(grad_out=torch.zeros(3, 8, dtype=torch.float16)), RuntimeError, "grad_out"),
    (dict(mean=torch.zeros(2, 1)), RuntimeError, "mean"),
    (dict(rstd=torch.zeros(3, 2)), RuntimeError, "rstd"),
    (dict(rstd=torch.zeros(3, 1, dtype=torch.int64)), NotImplementedError, "rstd"),
    (dict(weight=torch.ones(7)), RuntimeError, "weight"),
    (dict(weight=None), RuntimeError, "weight is None"),
    (dict(bias=None), RuntimeError, "bias is None"),
    (dict(weight=torch.ones(8, dtype=torch.float64)), RuntimeError, "same dtype"),
    (dict(input=torch.zeros(3, 8, dtype=torch.int32), grad_out=torch.zeros(3, 8, dtype=torch.int32)), NotImplementedError, "int32"),
])
def test_layer_norm_backward_refusals(change, error, match):
    with pytest.raises(error, match=match):
        ops.native_layer_norm_backward(**ln_args(**change))


@pytest.mark.parametrize("x,w,act,error,match", [
    (torch.zeros(2, 8), torch.zeros(6, 8), "tanh", ValueError, "activation"),
    (torch.zeros(2, 8), torch.zeros(5, 8), "silu", RuntimeError, "gate rows"),
    (torch.zeros(2, 8), torch.zeros(6, 8, 1), "silu", RuntimeError, "gate rows"),
    (torch.zeros(2, 7), torch.zeros(6, 8), "silu", RuntimeError, "cannot be multiplied"),
    (torch.zeros(()), torch.zeros(6, 1), "silu", RuntimeError, "cannot be multiplied"),
    (torch.zeros(2, 8).half(), torch.zeros(6, 8), "silu", RuntimeError, "same dtype"),
    (torch.zeros(2, 8, dtype=torch.int8), torch.zeros(6, 8, dtype=torch.int8), "silu", NotImplementedError, "int8"),
])
def test_gated_linear_refusals(x, w, act, error, match):
    with pytest.raises(error, match=match):
        ops.gated_linear(x, w, act)
    with pytest.raises(error, match=match):
        ops.gated_linear_backward(torch.zeros(2, 3), x, w, torch.zeros(2, 6), act)


@pytest.mark.parametrize("dh,pre,match", [
    (torch.zeros(2, 4), torch.zeros(2, 6), "grad_out"), (torch.zeros(2, 3), torch.zeros(2, 3), "pre"),
    (torch.zeros(2, 3).half(), torch.zeros(2, 6), "grad_out"), (torch.zeros(2, 3), torch.zeros(2, 6).half(), "pre"),
    (torch.zeros(3, 3), torch.zeros(2, 6), "grad_out"),
])
def test_gated_linear_backward_refusals(dh, pre, match):
    with pytest.raises(RuntimeError, match=match):
        ops.gated_linear_backward(dh, torch.zeros(2, 8), torch.zeros(6, 8), pre)
    with pytest.raises(RuntimeError, match="output_mask"):
        ops.gated_linear_backward(torch.zeros(2, 3), torch.zeros(2, 8), torch.zeros(6, 8), torch.zeros(2, 6), "silu", (True,))


@pytest.mark.parametrize("x,res,p,rng,error,match", [
    (torch.zeros(4), None, -0.1, (0, 0), RuntimeError, "probability"),
    (torch.zeros(4), None, 1.1, (0, 0), RuntimeError, "probability"),
    (torch.zeros(4), None, float("nan"), (0, 0), RuntimeError, "probability"),
    (torch.zeros(4), torch.zeros(5), 0.1, (0, 0), RuntimeError, "residual"),
    (torch.zeros(4), torch.zeros(4).half(), 0.1, (0, 0), RuntimeError, "residual"),
    (torch.zeros(4), None, 0.1, (0,), RuntimeError, "rng"),
    (torch.zeros(4), None, 0.1, torch.zeros(2), RuntimeError, "rng"),
    (torch.zeros(4), None, 0.1, torch.zeros(3, dtype=torch.int64), RuntimeError, "rng"),
    (torch.zeros(4, dtype=torch.int32), None, 0.1, (0, 0), NotImplementedError, "int32"),
])
def test_dropout_refusals(x, res, p, rng, error, match):
    with pytest.raises(error, match=match):
        ops.dropout_add(x, res, p, rng)


@pytest.mark.skipif(torch.cuda.is_available(), reason="host-only behaviour")
def test_no_fallback_without_a_gpu():
    for call in (lambda: ops.native_layer_norm_backward(**ln_args()), lambda: ops.gated_linear(torch.zeros(2, 8), torch.zeros(6, 8)),
                 lambda: ops.gated_linear_backward(torch.zeros(2, 3), torch.zeros(2, 8), torch.zeros(6, 8), torch.zeros(2, 6)),
                 lambda: ops.dropout_add(torch.zeros(4), None, 0.1, (0, 0)), lambda: ops.dropout_add_backward(torch.zeros(4), 0.1, (0, 0))):
        with pytest.raises(RuntimeError, match="no GPU visible"):
            call()


def test_c_entry_points_check_their_arguments():
    """Validation comes before any launch; the pointers are never dereferenced."""
    lib, p = _lib.load(), 1 << 20

    def refused(rc, text):
        assert rc < 0 and text in lib.mi355_last_error(), (rc, lib.mi355_last_error())

    ln = lib.mi355_layer_norm_backward
    assert lib.mi355_layer_norm_backward_workspace_bytes(4, 8, _lib.F32) == 0    # one block holds it all
    need = lib.mi355_layer_norm_backward_workspace_bytes(4000, 8, _lib.F32)
    assert need > 0
    refused(ln(p, p, _lib.F32, p, p, p, _lib.F32, p, p, p, 4000, 8, p, need - 1, None), b"workspace")
    refused(ln(p, p, _lib.F32, p, p, p, _lib.F32, p, p, p, 4000, 8, None, need, None), b"workspace")
    refused(ln(p, p, _lib.F32, p, p, p, _lib.F32, p, p, p, 4000, 8, p + 4, need, None), b"workspace")
    refused(ln(None, p, _lib.F32, p, p, p, _lib.F32, p, p, p, 4, 8, p, need, None), b"NULL")
    refused(ln(p, p, _lib.F32, p, p, p, _lib.F32, p, p, p, -1, 8, p, need, None), b"negative")
    refused(ln(p, p, _lib.F32, p, p, p, _lib.F32, p, p, p, 0, 8, p, need, None), b"no rows")
    refused(ln(p, p, _lib.F32, p, p, p, _lib.BF16, p, p, p, 4, 8, p, need, None), b"no kernel")
    refused(ln(p, p, _lib.I32, p, p, p, _lib.I32, p, p, p, 4, 8, p, need, None), b"no kernel")
    refused(ln(p, p, _lib.F32, p, p, p, _lib.F32, p, p, p, 4, 1 << 28, p, 1 << 60, None), b"too large")
    assert ln(p, p, _lib.F32, p, p, p, _lib.F32, None, None, None, 4, 8, None, 0, None) == 0   # nothing wanted
    assert ln(None, None, _lib.F32, None, None, None, _lib.F32, p, None, None, 0, 8, None, 0, None) == 0
    assert lib.mi355_layer_norm_backward_workspace_bytes(0, 8, _lib.F32) == 0
    act = lib.mi355_gated_act
    refused(act(p, p, _lib.F32, 4, 8, 3, None), b"activation")
    refused(act(None, p, _lib.F32, 4, 8, 0, None), b"NULL")
    refused(act(p, p, _lib.BF16, 4, 8, 0, None), b"unsupported")
    refused(act(p, p, _lib.F32, -4, 8, 0, None), b"negative")
    pad = lib.mi355_pad_rows
    refused(pad(p, 8, 4, 8, p, 12, 2, None), b"rows of 12")
    refused(pad(p, 8, 4, 8, p, 16, 8, None), b"of 8 bytes")
    refused(pad(p, 7, 4, 8, p, 16, 2, None), b"extents")
    refused(pad(p, 16, 4, 16, p, 8, 2, None), b"extents")
    refused(pad(p, 8, 4, 8, p + 8, 16, 2, None), b"misaligned")
    refused(pad(None, 8, 4, 8, p, 16, 2, None), b"NULL")
    assert pad(None, 8, 0, 8, None, 16, 2, None) == 0
    fwd = lib.mi355_gated_linear
    refused(fwd(p, 64, p, 64, p, None, 4, 8, 64, 3, _lib.BF16, None), b"activation")
    refused(fwd(None, 64, p, 64, p, None, 4, 8, 64, 0, _lib.BF16, None), b"NULL")
    refused(fwd(p, 63, p, 64, p, None, 4, 8, 64, 0, _lib.BF16, None), b"overlap")
    refused(fwd(p, 64, p, 0, p, None, 4, 8, 64, 0, _lib.BF16, None), b"overlap")
    refused(fwd(p, 64, p, 64, p, None, 4, -8, 64, 0, _lib.BF16, None), b"negative")
    for rows, K, dtype in ((33, 64, _lib.F32), (5, 7, _lib.F32), (9, 64, _lib.F64), (4, 64, _lib.I8), (4, 64, _lib.I32), (65, 63, _lib.BF16), (65, 72, _lib.F16), (5, 7, _lib.BF16),
                           (4, 0, _lib.BF16)):
        assert fwd(p, K, p, K, p, None, rows, 8, K, 0, dtype, None) == -2     # unsupported, nothing launched
    assert fwd(None, 64, None, 64, None, None, 0, 8, 64, 0, _lib.BF16, None) == 0
    back, size = lib.mi355_gated_linear_backward, lib.mi355_gated_linear_backward_workspace_bytes
    need = size(4, 8, 64, _lib.F32)
    assert need > 0 and size(0, 8, 64, _lib.F32) == 0 and size(4, 8, 64, _lib.U8) == 0
    refused(back(p, p, 64, p, 64, p, p, p, 4, 8, 64, -1, _lib.F32, p, need, None), b"activation")
    refused(back(p, p, 64, p, 64, None, p, p, 4, 8, 64, 0, _lib.F32, p, need, None), b"NULL")
    refused(back(p, p, 60, p, 64, p, p, p, 4, 8, 64, 0, _lib.F32, p, need, None), b"overlap")
    refused(back(p, p, 64, p, 64, p, p, p, 4, 8, 64, 0, _lib.F32, p, 16, None), b"workspace")
    refused(back(p, p, 64, p, 64, p, p, p, 4, 8, 64, 0, _lib.F32, p + 8, need, None), b"workspace")
    refused(back(p, p, 64, p, 64, p, p, p, 4, 8, 64, 0, _lib.F32, None, need, None), b"workspace")
    refused(back(p, p, 64, p, 64, p, p, p, 4, 8, 64, 0, _lib.U8, p, need, None), b"unsupported")
    refused(back(p, p, 64, p, 64, p, p, p, 0, 8, 64, 0, _lib.F32, p, need, None), b"empty")
    refused(back(p, p, 64, p, 64, p, p, p, 4, 8, -64, 0, _lib.F32, p, need, None), b"negative")
    assert back(None, None, 64, None, 64, None, None, None, 4, 8, 64, 0, _lib.F32, None, 0, None) == 0
    drop = lib.mi355_dropout_add
    refused(drop(p, None, _lib.F32, 1.5, None, 0, 0, p, 4, None), b"[0, 1]")
    refused(drop(p, None, _lib.F32, float("nan"), None, 0, 0, p, 4, None), b"[0, 1]")
    refused(drop(None, None, _lib.F32, 0.5, None, 0, 0, p, 4, None), b"NULL")
    refused(drop(p, None, _lib.F32, 0.5, p + 4, 0, 0, p, 4, None), b"aligned")
    refused(drop(p, None, _lib.I64, 0.5, None, 0, 0, p, 4, None), b"unsupported")
    refused(drop(p, None, _lib.F32, 0.5, None, 0, 0, p, -4, None), b"negative")
    assert drop(None, None, _lib.F32, 0.5, None, 0, 0, None, 0, None) == 0


# ---- the oracle ------------------------------------------------------------------------
def test_philox_known_answers():
    """Known-answer vectors published with the generator."""
    assert ref.philox4x32_10((0, 0, 0, 0), (0, 0)) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    f = 0xFFFFFFFF
    assert ref.philox4x32_10((f, f, f, f), (f, f)) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]


def test_dropout_keep_rate():
    for p in (0.1, 0.5):
        n = 40000
        kept = ref.dropout_keep(n, p, 1234, 77).sum().item()
        assert abs(kept - n * (1 - p)) < 5 * (n * p * (1 - p)) ** 0.5  # five standard deviations
    assert ref.dropout_keep(100, 0.0, 1, 0).all() and not ref.dropout_keep(100, 1.0, 1, 0).any()


def differences(f, x, step=1e-6):
    g = torch.zeros_like(x)
    for i in range(x.numel()):
        up, down = x.clone(), x.clone()
        up.view(-1)[i] += step
        down.view(-1)[i] -= step
        g.view(-1)[i] = (f(up) - f(down)) / (2 * step)
    return g


def test_layer_norm_formula_against_differences():
    gen = torch.Generator().manual_seed(3)
    x, dy = torch.randn(4, 6, generator=gen).double(), torch.randn(4, 6, generator=gen).double()
    w, b = torch.randn(6, generator=gen).double(), torch.randn(6, generator=gen).double()

    def loss(x, w, b):
        mu = x.mean(1, keepdim=True)
        return (((x - mu) / torch.sqrt((x - mu).square().mean(1, keepdim=True) + 1e-5) * w + b) * dy).sum().item()

    mean = x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt((x - mean).square().mean(1, keepdim=True) + 1e-5)
    (dx, dw, db), _ = ref.layer_norm_backward(dy, x, mean, rstd, w, 4, 6)
    for got, want in ((dx, differences(lambda t: loss(t, w, b), x)), (dw, differences(lambda t: loss(x, t, b), w)),
                      (db, differences(lambda t: loss(x, w, t), b))):
        assert torch.allclose(got, want, rtol=1e-6, atol=1e-7)


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_gated_formula_against_differences(act):
    gen = torch.Generator().manual_seed(4)
    x, w, dh = (torch.randn(*s, generator=gen).double() for s in ((3, 5), (8, 5), (3, 4)))

    def loss(x, w):
        return (ref.gated_linear(x, w, act)[0][0] * dh).sum().item()

    dpre = ref.gated_pre_backward(dh, ref.gated_linear(x, w, act)[0][1], act)
    assert torch.allclose(dpre @ w, differences(lambda t: loss(t, w), x), rtol=1e-6, atol=1e-7)
    assert torch.allclose(dpre.t() @ x, differences(lambda t: loss(x, t), w), rtol=1e-6, atol=1e-7)


def test_gated_backward_workspace_covers_every_alignment():
    """The size a caller asks for covers what any alignment of the operands takes (a call with less is refused)."""
    lib, p = _lib.load(), 1 << 20
    for M, F, K, dtype in ((64, 64, 64, _lib.BF16), (65, 33, 77, _lib.F16), (300, 1000, 768, _lib.BF16), (5, 3, 7, _lib.F32), (7, 9, 11, _lib.F64)):
        full = lib.mi355_gated_linear_backward_workspace_bytes(M, F, K, dtype)
        es = 2 if dtype in (_lib.F16, _lib.BF16) else 4 if dtype == _lib.F32 else 8
        assert full >= 2 * M * F * es and full % 256 == 0
        for x_off, w_off in ((0, 0), (es, 0), (0, es), (es, es)):
            for dx, dw in ((p, p), (p, None), (None, p)):
                rc = lib.mi355_gated_linear_backward(p, p + x_off, K, p + w_off, K, p, dx, dw, M, F, K, 0, dtype, p, 0, None)
                need = int(re.search(rb"workspace of (\d+) bytes", lib.mi355_last_error()).group(1))
                assert rc == -1 and 0 < need <= full, (M, F, K, dtype, need, full)
