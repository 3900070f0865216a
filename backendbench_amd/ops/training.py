"""Operators of a training step: layer norm's backward pass, the gated linear projection of a feed-forward block with
its backward pass, and dropout from a counter-based generator with the residual add.

Like the ATen overloads beside them these are kernels, not autograd nodes: they return plain results, and a gradient is
a call of the operator that computes it.  Arguments are checked before anything touches the GPU.
"""

import torch

from .. import _lib
from ._common import cast, copy_into, dense, launch, new_dense, new_result, on_gpu, prod, try_launch
from .elementwise import _store_result as store_result
from .elementwise import tuple_out_variant
from .matmul import _gemm

_FLOATS = (torch.float32, torch.float16, torch.bfloat16, torch.float64)
_HALF = (torch.bfloat16, torch.float16)


def _need_float(t, what):
    if t.dtype not in _FLOATS:
        raise NotImplementedError(f"mi355 backend: {what} on {t.dtype} is not supported")


def _ptr(t):
    return None if t is None else t.data_ptr()


# ---- layer norm, backward ------------------------------------------------------------------------------------------
def native_layer_norm_backward(grad_out, input, normalized_shape, mean, rstd, weight, bias, output_mask):
    """aten.native_layer_norm_backward.default -> (grad_input, grad_weight, grad_bias), None where output_mask is False.

    mean and rstd are what native_layer_norm returned; grad_weight and grad_bias have the dtype of weight and bias."""
    k, shape = len(normalized_shape), input.shape
    if k == 0 or k > len(shape) or shape[len(shape) - k :] != tuple(normalized_shape):
        raise RuntimeError(
            f"Given normalized_shape={list(normalized_shape)}, expected input with shape "
            f"[*, {', '.join(str(s) for s in normalized_shape)}], but got input of size{list(shape)}")
    _need_float(input, "layer norm")
    if grad_out.shape != shape:
        raise RuntimeError(f"Expected grad_out of the input's shape {list(shape)}, but got {list(grad_out.shape)}")
    if grad_out.dtype != input.dtype:
        raise RuntimeError(f"Expected grad_out of the input's dtype {input.dtype}, but got {grad_out.dtype}")
    M = prod(shape[: len(shape) - k])
    for name, s in (("mean", mean), ("rstd", rstd)):
        if s.numel() != M:
            raise RuntimeError(f"Expected {name} to hold {M} values, one per row, but got {s.numel()}")
        _need_float(s, name)
    for name, p, wanted in (("weight", weight, output_mask[1]), ("bias", bias, output_mask[2])):
        if p is None:
            if wanted:
                raise RuntimeError(f"the gradient of {name} was asked for, but {name} is None")
        elif p.shape != tuple(normalized_shape):
            raise RuntimeError(f"Expected {name} to be of same shape as normalized_shape, but got {name} of shape "
                               f"{list(p.shape)} and normalized_shape = {list(normalized_shape)}")
        else:
            _need_float(p, name)
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise RuntimeError("weight and bias must have the same dtype")
    return _layer_norm_backward(grad_out, input, mean, rstd, weight, bias, M, tuple(normalized_shape), output_mask)


_ln_workspace = None


@on_gpu
def _layer_norm_backward(grad_out, input, mean, rstd, weight, bias, M, normalized_shape, mask):
    global _ln_workspace
    N = prod(normalized_shape)
    dtype, device = input.dtype, input.device
    w_given = weight.dtype if weight is not None else bias.dtype if bias is not None else dtype
    dx = new_result(input.shape, dtype, device) if mask[0] else None
    dw = new_result(normalized_shape, w_given, device) if mask[1] else None
    db = new_result(normalized_shape, w_given, device) if mask[2] else None
    if M == 0 or N == 0 or not (mask[0] or mask[1] or mask[2]):
        for g in (dw, db):
            if g is not None:
                g.zero_()
        return dx, dw, db
    # the kernels take parameters of the rows' dtype, or fp32 beside bf16 / f16 rows
    w_dtype = w_given
    if w_given != dtype:
        w_dtype = torch.float32 if dtype in _HALF else dtype  # (never through a type narrower than both)
    stat_dtype = torch.float64 if dtype == torch.float64 else torch.float32
    x, dy = dense(input), dense(grad_out)
    mu, rs = dense(cast(mean, stat_dtype)), dense(cast(rstd, stat_dtype))
    w = dense(cast(weight, w_dtype)) if weight is not None else None
    own_dw, own_db = dw, db  # what the kernel writes
    if w_given != w_dtype:
        own_dw = new_dense(normalized_shape, w_dtype, device) if mask[1] else None
        own_db = new_dense(normalized_shape, w_dtype, device) if mask[2] else None
    code = _lib.DTYPE[dtype]
    if _ln_workspace is None:
        _ln_workspace = _lib.load().mi355_layer_norm_backward_workspace_bytes
    ws_bytes = _ln_workspace(M, N, code)
    ws = new_dense((ws_bytes,), torch.uint8, device) if ws_bytes else None
    launch("mi355_layer_norm_backward", dy.data_ptr(), x.data_ptr(), code, mu.data_ptr(), rs.data_ptr(), _ptr(w),
           _lib.DTYPE[w_dtype], _ptr(dx), _ptr(own_dw), _ptr(own_db), M, N, _ptr(ws), ws_bytes)
    if dw is not own_dw:
        copy_into(dw, own_dw)
    if db is not own_db:
        copy_into(db, own_db)
    return dx, dw, db


_out_all = tuple_out_variant(native_layer_norm_backward, 3)


def native_layer_norm_backward_out(grad_out, input, normalized_shape, mean, rstd, weight, bias, output_mask, *, out0, out1, out2):
    """aten.native_layer_norm_backward.out; an out tensor whose output_mask entry is False is left as it is."""
    args = (grad_out, input, normalized_shape, mean, rstd, weight, bias, output_mask)
    if all(output_mask):
        return _out_all(*args, out0=out0, out1=out1, out2=out2)
    results = native_layer_norm_backward(*args)
    return tuple(o if r is None else store_result(o, r) for o, r in zip((out0, out1, out2), results))


# ---- gated linear projection ---------------------------------------------------------------------------------------
_ACTIVATIONS = {"silu": _lib.SILU, "gelu": _lib.GELU, "gelu_tanh": _lib.GELU_TANH}


def _check_gated(input, weight, activation):
    if activation not in _ACTIVATIONS:
        raise ValueError(f"activation must be one of {', '.join(_ACTIVATIONS)}, got {activation!r}")
    _need_float(input, "gated_linear")
    if weight.dtype != input.dtype:
        raise RuntimeError(f"expected input and weight to have the same dtype, but got: {input.dtype} != {weight.dtype}")
    if weight.dim() != 2 or weight.shape[0] % 2:
        raise RuntimeError(f"weight must be [2 * features, in_features] (gate rows, then up rows), got {list(weight.shape)}")
    if input.dim() == 0 or input.shape[-1] != weight.shape[1]:
        raise RuntimeError(f"input {list(input.shape)} and weight {list(weight.shape)} cannot be multiplied: the last dimension of "
                           "input must be weight's second")


def gated_linear(input, weight, activation="silu", save_pre=False):
    """act(input @ weight[:F].T) * (input @ weight[F:].T) over the last dimension of input; weight is [2F, K].

    activation: "silu", "gelu" (by the error function) or "gelu_tanh".  Products are accumulated in fp32 (fp64 for
    fp64) and not rounded before the activation.  save_pre: also return the pre-activations [..., 2F] in the input's
    dtype, which gated_linear_backward takes; the one rounding between the two passes."""
    _check_gated(input, weight, activation)
    return _gated_linear(input, weight, _ACTIVATIONS[activation], save_pre)


def _rows_of(t):
    """`t` [R, K] itself when its rows are unit-stride and do not overlap, else a dense copy; one row K apart from the next
    (a tensor's own stride along a dimension of 1 says nothing: a column's transpose has 1)."""
    if t.shape[0] == 1 and t.stride() != (t.shape[1], 1):
        return dense(t).as_strided((1, t.shape[1]), (t.shape[1], 1))
    return t if t.stride(1) == 1 and t.stride(0) >= t.shape[1] else dense(t)


def _padded(t, columns):
    """A copy of `t` [R, K] in aligned rows of `columns` elements, zeros behind the K that are there (a product's terms 0 * 0)."""
    out = new_dense((t.shape[0], columns), t.dtype, t.device)
    launch("mi355_pad_rows", t.data_ptr(), t.stride(0), t.shape[0], t.shape[1], out.data_ptr(), columns, t.element_size())
    return out


_WIDE_ROWS = {torch.float32: 32, torch.float64: 8}  # mi355_gated_linear takes up to this many


@on_gpu
def _gated_linear(input, weight, act, save_pre):
    lead, K = input.shape[:-1], input.shape[-1]
    M, F = prod(lead), weight.shape[0] // 2
    dtype, device = input.dtype, input.device
    if M == 0 or F == 0 or K == 0:  # (no terms: pre = 0 and act(0) = 0)
        h = torch.zeros((*lead, F), dtype=dtype, device=device)
        return (h, torch.zeros((*lead, 2 * F), dtype=dtype, device=device)) if save_pre else h
    code = _lib.DTYPE[dtype]
    h = new_dense((*lead, F), dtype, device)
    x = _rows_of(input) if input.dim() == 2 else dense(input).view(M, K)
    weight = _rows_of(weight)
    if dtype in _HALF or M <= _WIDE_ROWS[dtype]:
        pre = new_dense((*lead, 2 * F), dtype, device) if save_pre else None

        def fused(attempt, x, weight, K):
            return attempt("mi355_gated_linear", x.data_ptr(), x.stride(0), weight.data_ptr(), weight.stride(0), h.data_ptr(), _ptr(pre),
                           M, F, K, act, code)

        done = fused(try_launch, x, weight, K)
        if not done and dtype in _HALF:  # rows that no kernel takes: padded ones
            Kp = max((K + 127) // 128 * 128, 256)
            fused(launch, _padded(x, Kp), _padded(weight, Kp), Kp)
            done = True
        if done:
            return (h, pre) if save_pre else h
    if dtype == torch.float32 and (K % 16 or any(t.data_ptr() % 16 or t.stride(0) % 4 for t in (x, weight))):
        # rows the fp32 matrix instructions' kernel takes; the product alone: [64, 5001] x 2 * 5001 180 -> 131 us with the copies, [64, 1001] x 2 * 771 21 -> 17,
        # [64, 4096] x 2 * 5504 and [512, 2048] x 2 * 2752 with rows K + 1 apart 363 -> 133 and 236 -> 131
        Kp = (K + 63) // 64 * 64
        x, weight = _padded(x, Kp), _padded(weight, Kp)
    pre = _gemm(x, weight.t(), None, 1.0, 0.0)
    launch("mi355_gated_act", pre.data_ptr(), h.data_ptr(), code, M, F, act)
    return (h, pre.view(*lead, 2 * F)) if save_pre else h


def gated_linear_backward(grad_out, input, weight, pre, activation="silu", output_mask=(True, True)):
    """Gradients of gated_linear -> (grad_input, grad_weight), None where output_mask is False.

    pre: the pre-activations gated_linear(..., save_pre=True) returned.  The gradient of pre is computed in fp32 and
    rounded once to the input's dtype: it is the operand of the two matrix products, which accumulate in fp32.  In f16
    that is also a bound on its range: a gradient of pre beyond 65504 becomes infinite, and with it its row of grad_input and its
    row of grad_weight - nothing else - which is what a loss scale's check for infinities looks for."""
    _check_gated(input, weight, activation)
    F = weight.shape[0] // 2
    lead = list(input.shape[:-1])
    for name, t, last in (("grad_out", grad_out, F), ("pre", pre, 2 * F)):
        if list(t.shape) != lead + [last]:
            raise RuntimeError(f"Expected {name} of shape {lead + [last]}, but got {list(t.shape)}")
        if t.dtype != input.dtype:
            raise RuntimeError(f"Expected {name} of the input's dtype {input.dtype}, but got {t.dtype}")
    if len(output_mask) != 2:
        raise RuntimeError(f"output_mask must have 2 entries, got {len(output_mask)}")
    return _gated_linear_backward(grad_out, input, weight, pre, _ACTIVATIONS[activation], output_mask)


@on_gpu
def _gated_linear_backward(grad_out, input, weight, pre, act, mask):
    K, F = weight.shape[1], weight.shape[0] // 2
    M = prod(input.shape[:-1])
    dtype, device = input.dtype, input.device
    if M == 0 or F == 0 or K == 0 or not (mask[0] or mask[1]):
        return (torch.zeros_like(input) if mask[0] else None), (torch.zeros_like(weight) if mask[1] else None)
    dh, p = dense(grad_out), dense(pre)
    x = _rows_of(input) if input.dim() == 2 else dense(input).view(M, K)
    w = _rows_of(weight)
    dx = new_dense(input.shape, dtype, device) if mask[0] else None
    dw = new_dense(weight.shape, dtype, device) if mask[1] else None
    code = _lib.dtype_code(dtype)
    ws_bytes = _lib.load().mi355_gated_linear_backward_workspace_bytes(M, F, K, code)
    ws = new_dense((ws_bytes,), torch.uint8, device)
    launch("mi355_gated_linear_backward", dh.data_ptr(), x.data_ptr(), x.stride(0), w.data_ptr(), w.stride(0), p.data_ptr(),
           _ptr(dx), _ptr(dw), M, F, K, act, code, ws.data_ptr(), ws_bytes)
    return dx, dw


# ---- dropout with a residual ---------------------------------------------------------------------------------------
def dropout_counters(numel):
    """Counters a dropout_add over `numel` elements uses up: the next call's offset is this one's plus that."""
    return (numel + 7) // 8


def _check_dropout(x, p, rng):
    _need_float(x, "dropout")
    if not 0.0 <= p <= 1.0:
        raise RuntimeError(f"dropout probability has to be between 0 and 1, but got {p}")
    if isinstance(rng, torch.Tensor):
        if rng.dtype != torch.int64 or list(rng.shape) != [2]:
            raise RuntimeError(f"rng must hold two int64 values, (seed, offset), got {rng.dtype} {list(rng.shape)}")
    elif len(rng) != 2:
        raise RuntimeError(f"rng must hold two values, (seed, offset), got {len(rng)}")


def dropout_add(input, residual, p, rng):
    """residual + dropout(input, p) (residual None: dropout(input, p)); the mask is never stored.

    rng: (seed, offset), two Python integers or an int64 tensor of two.  An int64 tensor on the GPU is read by the
    kernel, so a captured graph draws anew once the program has advanced it.  Element i of input (in row-major order,
    whatever its strides) takes the i % 8-th 16 bits of Philox-4x32-10 at counter offset + i // 8 under key seed and is
    dropped when they are below t = round(p * 65536), halves to the even neighbour; what is kept is scaled by
    65536 / (65536 - t), which makes the expectation exact for the p that 16 bits can hold.  Advance the offset by dropout_counters(input.numel())."""
    _check_dropout(input, p, rng)
    if residual is not None and (residual.shape != input.shape or residual.dtype != input.dtype):
        raise RuntimeError(f"Expected residual of the input's shape and dtype, {list(input.shape)} {input.dtype}, but got "
                           f"{list(residual.shape)} {residual.dtype}")
    return _dropout_add(input, residual, float(p), rng)


def dropout_add_backward(grad_out, p, rng):
    """Gradient of dropout_add with respect to its input, from the same p and rng (the residual's is grad_out itself)."""
    _check_dropout(grad_out, p, rng)
    return _dropout_add(grad_out, None, float(p), rng)


def _int64(v):
    return (int(v) + 2 ** 63) % 2 ** 64 - 2 ** 63


@on_gpu
def _dropout_add(input, residual, p, rng):
    out = new_dense(input.shape, input.dtype, input.device)
    if input.numel() == 0:
        return out
    x = dense(input)
    res = dense(residual) if residual is not None else None
    words, seed, offset = None, 0, 0
    if isinstance(rng, torch.Tensor):
        words = dense(rng)
    else:
        seed, offset = (_int64(v) for v in rng)
    launch("mi355_dropout_add", x.data_ptr(), _ptr(res), _lib.DTYPE[x.dtype], p, _ptr(words), seed, offset, out.data_ptr(), x.numel())
    return out
