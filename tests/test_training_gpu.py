"""The training operators on the GPU against the float64 definitions (oracle/training_ref.py).

Tolerances are sums of rounding errors: half a step of the output's type at the exact value, plus a count of fp32 (fp64)
roundings u = 2^-24 (2^-53) against the sum of the terms' absolute values.  A sum of L terms held in several partial
sums is charged 64 + L / 64 roundings (no kernel adds more than L / 64 terms in a row, and 64 covers the joins and the
term's own arithmetic); a matrix product, whose matrix instructions do not say in which order they add, 64 + K / 8."""

import pytest
import torch

import backendbench_amd
from backendbench_amd import _lib, ops
from oracle import training_ref as ref

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16, torch.float64]
HALF = (torch.float16, torch.bfloat16)


def unit(dtype):
    return 2.0 ** -53 if dtype == torch.float64 else 2.0 ** -24


def half_step(dtype, want):
    """Half a step of `dtype` at `want`; under the normal range the step of the smallest normal."""
    return want.abs().clamp_min(torch.finfo(dtype).tiny) * (torch.finfo(dtype).eps / 2)


def check(got, want, slack, what):
    """|got - want| <= half a step of got's type + slack, everywhere."""
    assert got.shape == want.shape, (what, got.shape, want.shape)
    err, tol = (got.double() - want).abs(), half_step(got.dtype, want) + slack
    bad = ~(err <= tol)
    if bad.any():
        i = int((err / tol).flatten().nan_to_num(float("inf")).argmax())
        raise AssertionError(f"{what} ({got.dtype}): {int(bad.sum())} of {bad.numel()} off; worst at {i}: got {got.flatten()[i].item()!r}, "
                             f"exact {want.flatten()[i].item()!r}, allowed {tol.flatten()[i].item():.3e}")


def randn(gen, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ---- layer norm, backward --------------------------------------------------------------
def ln_case(rows, cols, dtype, wdtype, seed, weight=True):
    g = generator(seed)
    x = randn(g, rows, cols, dtype=dtype, scale=2.0) + randn(g, cols, dtype=dtype)
    dy = randn(g, rows, cols, dtype=dtype, scale=0.1)
    stat = torch.float64 if dtype == torch.float64 else torch.float32
    xd = x.double()
    mean = xd.mean(1, keepdim=True)
    rstd = torch.rsqrt((xd - mean).square().mean(1, keepdim=True) + 1e-5)
    w = randn(g, cols, dtype=wdtype) if weight else None
    b = randn(g, cols, dtype=wdtype) if weight else None
    return dy, x, mean.to(stat), rstd.to(stat), w, b


def ln_check(got, dy, x, mean, rstd, w, rows, cols, what):
    want, scale = ref.layer_norm_backward(dy, x, mean, rstd, w, rows, cols)
    u = unit(x.dtype)
    for i, (length, shape) in enumerate(((cols, (rows, cols)), (rows, (cols,)), (rows, (cols,)))):
        if got[i] is not None:
            check(got[i].reshape(shape), want[i], (64 + length / 64) * u * scale[i], f"{what} output {i}")


SIZES = [(1, 1), (1, 7), (3, 64), (5, 130), (257, 128), (33, 768), (64, 1000), (17, 1001), (7, 4096), (300, 4104), (129, 2048),
         (2, 16384), (3, 16390), (1, 100001), (2000, 2), (1025, 512), (70000, 8), (1031, 264), (5000, 96)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", SIZES)
def test_layer_norm_backward(rows, cols, dtype):
    case = ln_case(rows, cols, dtype, dtype, rows + cols)
    got = ops.native_layer_norm_backward(case[0], case[1], [cols], *case[2:], [True] * 3)
    assert [t.dtype for t in got] == [dtype] * 3
    ln_check(got, *case[:5], rows, cols, f"[{rows}, {cols}]")


@pytest.mark.parametrize("dtype,wdtype", [(torch.bfloat16, torch.float32), (torch.float16, torch.float32), (torch.bfloat16, torch.float16),
                                          (torch.float32, torch.bfloat16), (torch.float32, torch.float64), (torch.float64, torch.float32)])
def test_layer_norm_backward_mixed_parameter_types(dtype, wdtype):
    rows, cols = 65, 776
    dy, x, mean, rstd, w, b = ln_case(rows, cols, dtype, wdtype, 5)
    w, b = w.float().bfloat16().to(wdtype), b  # values every one of these types holds
    got = ops.native_layer_norm_backward(dy, x, [cols], mean, rstd, w, b, [True] * 3)
    assert [t.dtype for t in got] == [dtype, wdtype, wdtype]
    want, scale = ref.layer_norm_backward(dy, x, mean, rstd, w, rows, cols)
    u = max(unit(dtype), 2.0 ** -24 if wdtype != torch.float64 else 0.0)
    for i in range(3):
        # a gradient wider than the rows is held in the rows' arithmetic, fp32, and widened at the end
        check(got[i], want[i], 77 * u * scale[i], f"{dtype} {wdtype} output {i}")


@pytest.mark.parametrize("rows,cols", [(40, 320), (9, 1001), (2100, 1024)])
@pytest.mark.parametrize("mask", [(True, False, False), (False, True, False), (False, False, True), (False, True, True), (True, False, True)])
def test_layer_norm_backward_masks(rows, cols, mask):
    case = ln_case(rows, cols, torch.bfloat16, torch.bfloat16, 6)
    got = ops.native_layer_norm_backward(case[0], case[1], [cols], *case[2:], list(mask))
    assert tuple(t is not None for t in got) == mask
    ln_check(got, *case[:5], rows, cols, str(mask))
    assert ops.native_layer_norm_backward(case[0], case[1], [cols], *case[2:], [False] * 3) == (None, None, None)


@pytest.mark.parametrize("rows,cols", [(40, 320), (3, 33000), (513, 129)])
def test_layer_norm_backward_without_weight(rows, cols):
    dy, x, mean, rstd, _, _ = ln_case(rows, cols, torch.float32, torch.float32, 7, weight=False)
    got = ops.native_layer_norm_backward(dy, x, [cols], mean, rstd, None, None, [True, False, False])
    ln_check(got, dy, x, mean, rstd, None, rows, cols, "no weight")
    bias = torch.zeros(cols, device="cuda")
    got = ops.native_layer_norm_backward(dy, x, [cols], mean, rstd, None, bias, [True, False, True])
    ln_check(got, dy, x, mean, rstd, None, rows, cols, "bias only")


def test_layer_norm_backward_shapes_strides_and_empties():
    g = generator(8)
    base, dbase = randn(g, 6, 40, 5, dtype=torch.bfloat16), randn(g, 5, 6, 40, dtype=torch.bfloat16)
    x, dy = base.permute(2, 0, 1), dbase
    w, b = randn(g, 40, 6, dtype=torch.bfloat16).t(), randn(g, 6, 40, dtype=torch.bfloat16)
    mean, rstd = x.float().mean((1, 2), keepdim=True), torch.rsqrt(x.float().var((1, 2), unbiased=False, keepdim=True) + 1e-5)
    got = ops.native_layer_norm_backward(dy, x, [6, 40], mean, rstd, w, b, [True] * 3)
    assert got[0].shape == x.shape and got[1].shape == w.shape
    want, scale = ref.layer_norm_backward(dy, x.contiguous(), mean, rstd, w.contiguous(), 5, 240)
    for i, shape in enumerate(((5, 240), (240,), (240,))):
        check(got[i].reshape(shape), want[i], 70 * 2.0 ** -24 * scale[i], f"permuted {i}")
    # rows whose storage starts off a 16-byte boundary
    flat, dflat = randn(g, 20 * 256 + 1, dtype=torch.float16)[1:], randn(g, 20 * 256 + 3, dtype=torch.float16)[3:]
    x, dy = flat.view(20, 256), dflat.view(20, 256)
    mean, rstd = x.float().mean(1, keepdim=True), torch.rsqrt(x.float().var(1, unbiased=False, keepdim=True) + 1e-5)
    w = randn(g, 257, dtype=torch.float16)[1:]
    got = ops.native_layer_norm_backward(dy, x, [256], mean, rstd, w, w, [True] * 3)
    ln_check(got, dy, x, mean, rstd, w, 20, 256, "off alignment")
    # no rows: zero parameter gradients; no columns: empty everything
    e = torch.empty(0, 16, device="cuda")
    s = torch.empty(0, 1, device="cuda")
    dx, dw, db = ops.native_layer_norm_backward(e, e, [16], s, s, torch.ones(16, device="cuda"), torch.ones(16, device="cuda"), [True] * 3)
    assert dx.shape == (0, 16) and dw.tolist() == [0.0] * 16 and db.tolist() == [0.0] * 16
    e, s, z = torch.empty(4, 0, device="cuda"), torch.zeros(4, 1, device="cuda"), torch.empty(0, device="cuda")
    assert [t.numel() for t in ops.native_layer_norm_backward(e, e, [0], s, s, z, z, [True] * 3)] == [0, 0, 0]


def test_layer_norm_backward_infinities_stay_in_their_row():
    """A NaN or an infinity reaches its own row of dx and its columns' parameter gradients, and nothing else."""
    rows, cols = 300, 512
    case = list(ln_case(rows, cols, torch.float32, torch.float32, 9))
    clean = ops.native_layer_norm_backward(case[0], case[1], [cols], *case[2:], [True] * 3)
    case[0] = case[0].clone()
    case[0][41, 7] = float("inf")
    case[0][200, 300] = float("nan")
    got = ops.native_layer_norm_backward(case[0], case[1], [cols], *case[2:], [True] * 3)
    rows_ok = torch.ones(rows, dtype=torch.bool, device="cuda")
    rows_ok[[41, 200]] = False
    cols_ok = torch.ones(cols, dtype=torch.bool, device="cuda")
    cols_ok[[7, 300]] = False
    assert torch.equal(got[0][rows_ok], clean[0][rows_ok]) and not got[0][200].isfinite().any()
    for i in (1, 2):
        assert torch.equal(got[i][cols_ok], clean[i][cols_ok]) and not got[i][~cols_ok].isfinite().any()


@pytest.mark.parametrize("rows,cols", [(3, 100), (300, 520), (2, 777), (9, 5000), (2, 16384)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layer_norm_backward_infinite_weight(dtype, rows, cols):
    """An infinite weight in the last column gives what the formula gives: lanes behind the row's end do not multiply it by 0."""
    dy, x, mean, rstd, w, b = ln_case(rows, cols, dtype, dtype, 31)
    w[-1], dy[:, -1] = float("inf"), 1.0
    dx, dw, _ = ops.native_layer_norm_backward(dy, x, [cols], mean, rstd, w, b, [True] * 3)
    xhat, g = (x.double() - mean.double()) * rstd.double(), dy.double() * w.double()
    want = rstd.double() * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
    assert torch.equal(dx.isnan(), want.isnan()) and torch.equal(dx == -float("inf"), want == -float("inf"))
    assert dw.isfinite().all()


def test_layer_norm_backward_repeats_bit_for_bit():
    case = ln_case(4099, 1024, torch.bfloat16, torch.float32, 10)
    first = ops.native_layer_norm_backward(case[0], case[1], [1024], *case[2:], [True] * 3)
    for _ in range(3):
        again = ops.native_layer_norm_backward(case[0], case[1], [1024], *case[2:], [True] * 3)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_layer_norm_backward_slots_and_autograd(repo_root):
    """The folder tree: out= overload, and autograd of F.layer_norm under the dispatcher override."""
    rows, cols = 37, 768
    dy, x, mean, rstd, w, b = ln_case(rows, cols, torch.float32, torch.float32, 11)
    from backendbench_amd.backends import DirectoryBackend

    backend = DirectoryBackend(repo_root + "/generated_training_kernels")
    aten = torch.ops.aten.native_layer_norm_backward
    outs = [torch.full_like(t, 3.0) for t in (x, w, b)]
    res = backend[aten.out](dy, x, [cols], mean, rstd, w, b, [True] * 3, out0=outs[0], out1=outs[1], out2=outs[2])
    assert all(r is o for r, o in zip(res, outs))
    ln_check(outs, dy, x, mean, rstd, w, rows, cols, "out=")
    outs = [torch.full_like(t, 3.0) for t in (x, w, b)]
    backend[aten.out](dy, x, [cols], mean, rstd, w, b, [False, True, False], out0=outs[0], out1=outs[1], out2=outs[2])
    assert (outs[0] == 3.0).all() and (outs[2] == 3.0).all()
    ln_check([None, outs[1], None], dy, x, mean, rstd, w, rows, cols, "out= masked")
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    with backendbench_amd.BackendBench.enable(kernel_dir=repo_root + "/generated_kernels"):
        with backendbench_amd.BackendBench.enable(kernel_dir=repo_root + "/generated_training_kernels"):
            y = torch.nn.functional.layer_norm(leaves[0], [cols], leaves[1], leaves[2], 1e-5)
            grads = torch.autograd.grad(y, leaves, dy)
            assert torch.autograd.grad(torch.nn.functional.layer_norm(leaves[0], [cols]), leaves[:1], dy)[0].shape == x.shape
    ln_check(grads, dy, x, mean, rstd, w, rows, cols, "autograd")


# ---- gated linear projection -----------------------------------------------------------
def act_error(name, g, u):
    """fp32 roundings of act(g) against |act(g)|: the exponential's argument is rounded at |g| (|z| for tanh)."""
    z = g.abs() if name == "silu" else 0.5 * g * g if name == "gelu" else 1.6 * (g.abs() + 0.045 * g.abs() ** 3)
    return (32 + 4 * z) * u


def gated_forward_check(h, pre, x, w, act, what):
    (want_h, want_pre), scale = ref.gated_linear(x, w, act)
    u, K, F = unit(x.dtype), x.shape[1], w.shape[0] // 2
    dp = (64 + K / 8) * u * scale
    g, up = want_pre[:, :F], want_pre[:, F:]
    a = ref.activation(g, act)[0].abs()
    slack = dp[:, :F] * 1.2 * (up.abs() + dp[:, F:]) + dp[:, F:] * a + act_error(act, g, u) * a * up.abs()  # |act'| < 1.2
    slack = slack + 2.0 ** -126 * g.abs() * up.abs()  # an exponential under the smallest normal number may come out as zero
    check(h, want_h, slack, f"{what} h")
    if pre is not None:
        check(pre, want_pre, dp, f"{what} pre")


def gated_backward_check(got, dh, x, w, pre, act, what):
    u, F = unit(x.dtype), w.shape[0] // 2
    M, K = x.shape
    dpre = ref.gated_pre_backward(dh, pre, act)
    g, up = pre[:, :F].double(), pre[:, F:].double()
    terms = torch.cat([dh.double().abs() * up.abs() * (1 + g.abs()), dh.double().abs() * ref.activation(g, act)[0].abs()], 1)
    # dpre is rounded to the inputs' type once; its own arithmetic as in the forward
    edp = half_step(x.dtype, dpre) + act_error(act, torch.cat([g, g], 1), u) * terms
    # an exponential e (or erfc) under the smallest normal number is only right to 2^-126 absolutely (subnormal steps, or
    # zero in its place); |d gate| / e <= |dh up| (1 + g^2) and |d up| / e <= |dh g|, both under the factor here
    edp = edp + 2.0 ** -126 * (dh.double().abs() * (1 + up.abs()) * (1 + g * g)).repeat(1, 2)
    ad, ax, aw = dpre.abs() + edp, x.double().abs(), w.double().abs()
    if got[0] is not None:
        check(got[0], dpre @ w.double(), edp @ aw + (64 + 2 * F / 8) * u * (ad @ aw), f"{what} dx")
    if got[1] is not None:
        check(got[1], dpre.t().contiguous() @ x.double(), edp.t().contiguous() @ ax + (64 + M / 8) * u * (ad.t().contiguous() @ ax), f"{what} dw")


GATED = [(1, 1, 1), (1, 256, 64), (1, 4096, 1376), (2, 72, 40), (3, 1000, 24), (7, 2048, 344), (16, 512, 200), (17, 130, 33), (33, 768, 256),
         (48, 2048, 688), (64, 264, 129), (65, 1024, 96), (100, 771, 101), (128, 384, 128), (197, 768, 250), (256, 256, 128), (257, 640, 136),
         (300, 1001, 77), (512, 1152, 1000), (1030, 256, 264)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K,F", GATED)
def test_gated_linear(M, K, F, dtype):
    g = generator(M + K + F)
    act = ["silu", "gelu", "gelu_tanh"][(M + K + F) % 3]
    x, w = randn(g, M, K, dtype=dtype), randn(g, 2 * F, K, dtype=dtype, scale=K ** -0.5)
    h, pre = ops.gated_linear(x, w, act, save_pre=True)
    assert h.dtype == pre.dtype == dtype
    gated_forward_check(h, pre, x, w, act, f"{M}x{K}x{F} {act}")
    assert torch.equal(ops.gated_linear(x, w, act), h)  # keeping pre changes nothing
    dh = randn(g, M, F, dtype=dtype, scale=0.1)
    got = ops.gated_linear_backward(dh, x, w, pre, act)
    assert got[0].dtype == got[1].dtype == dtype
    gated_backward_check(got, dh, x, w, pre, act, f"{M}x{K}x{F} {act}")


@pytest.fixture
def gated_form():
    yield lambda value: _lib.set_knob("gated_form", value)
    _lib.set_knob("gated_form", None)


@pytest.mark.parametrize("form,M,K,F", [
    ("rows", 1, 2048, 40), ("rows", 16, 1016, 24), ("rows", 17, 2056, 23), ("rows", 64, 4104, 129), ("rows", 33, 8, 1), ("rows", 5, 5120, 8),
    ("dots", 1, 2048, 40), ("dots", 2, 1000, 129), ("dots", 1, 77, 9), ("dots", 2, 1331, 33), ("dots", 2, 4103, 1), ("dots", 2, 511, 4097),
    ("dots", 1, 513, 5000),
    ("tile128", 1, 64, 1), ("tile128", 130, 128, 70), ("tile128", 64, 192, 64), ("tile128", 300, 256, 129), ("tile128", 257, 448, 200),
    ("tile128", 128, 1024, 336),
    ("tile256", 1, 256, 1), ("tile256", 300, 384, 129), ("tile256", 257, 640, 128), ("tile256", 512, 1024, 264),
    ("tile256", 1000, 640, 4104)])
@pytest.mark.parametrize("dtype", HALF)
def test_gated_linear_forms(gated_form, form, M, K, F, dtype):
    """Every kernel form on shapes of the test's choosing: ragged and single tiles, short K loops, with and without pre."""
    g = generator(M + F)
    x, w = randn(g, M, K, dtype=dtype), randn(g, 2 * F, K, dtype=dtype, scale=K ** -0.5)
    act = ["silu", "gelu", "gelu_tanh"][F % 3]
    gated_form(form)
    h, pre = ops.gated_linear(x, w, act, save_pre=True)
    gated_forward_check(h, pre, x, w, act, f"{form} {M}x{K}x{F} {act}")
    assert torch.equal(ops.gated_linear(x, w, act), h)


@pytest.mark.parametrize("M,K,F", [(1, 1, 1), (1, 4096, 300), (2, 770, 5), (3, 255, 2049), (5, 513, 64), (8, 1027, 33), (9, 100, 33), (16, 4099, 17),
                                   (17, 257, 40), (33, 1000, 24), (64, 777, 40), (40, 263, 9), (5, 8, 16), (64, 9, 3), (12, 7, 30)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_gated_linear_few_rows_at_any_address(dtype, M, K, F):
    """Operands in odd columns of wider tensors, NaN around them."""
    g = generator(M * K + F)
    x, w = randn(g, M, K + 3, dtype=dtype), randn(g, 2 * F + 1, K + 5, dtype=dtype, scale=K ** -0.5)
    x[:, :1], x[:, K + 1:], w[:, :3], w[:, K + 3:], w[2 * F:] = (float("nan"),) * 5
    x, w = x[:, 1:K + 1], w[:2 * F, 3:K + 3]
    act = ["silu", "gelu", "gelu_tanh"][M % 3]
    h, pre = ops.gated_linear(x, w, act, save_pre=True)
    gated_forward_check(h, pre, x, w, act, f"{M}x{K}x{F} {act}")
    assert torch.equal(ops.gated_linear(x, w, act), h)


@pytest.mark.parametrize("M,K,F", [(1, 8, 1), (1, 2049, 9), (2, 511, 300), (7, 9, 65), (8, 768, 41), (9, 513, 7), (16, 1001, 130), (17, 100, 33)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_gated_linear_backward_few_rows(dtype, M, K, F):
    """Operands in odd columns of wider tensors, NaN around them; each gradient alone gives the same."""
    g = generator(M + K + F)
    x, w = randn(g, M, K + 3, dtype=dtype), randn(g, 2 * F + 1, K + 5, dtype=dtype, scale=K ** -0.5)
    x[:, :1], x[:, K + 1:], w[:, :3], w[:, K + 3:], w[2 * F:] = (float("nan"),) * 5
    x, w = x[:, 1:K + 1], w[:2 * F, 3:K + 3]
    pre, dh = randn(g, M, 2 * F, dtype=dtype), randn(g, M, F, dtype=dtype)
    act = ["silu", "gelu", "gelu_tanh"][M % 3]
    got = ops.gated_linear_backward(dh, x, w, pre, act)
    gated_backward_check(got, dh, x, w, pre, act, f"{M}x{K}x{F} {act}")
    dx, none = ops.gated_linear_backward(dh, x, w, pre, act, (True, False))
    assert none is None and torch.equal(dx, got[0])
    none, dw = ops.gated_linear_backward(dh, x, w, pre, act, (False, True))
    assert none is None and torch.equal(dw, got[1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_gated_linear_far_gates(act, dtype):
    """Gates from -90 to 90: the activation saturates without overflow, its gradient too."""
    M, F = 5, 361
    x = torch.eye(8, device="cuda", dtype=dtype)[:M]
    w = torch.zeros(2 * F, 8, device="cuda", dtype=dtype)
    w[:F, :M] = torch.linspace(-90, 90, F, device="cuda").to(dtype)[:, None]
    w[F:, :M] = 1.5
    h, pre = ops.gated_linear(x, w, act, save_pre=True)
    gated_forward_check(h, pre, x, w, act, act)
    dh = torch.ones(M, F, device="cuda", dtype=dtype)
    got = ops.gated_linear_backward(dh, x, w, pre, act)
    assert all(t.isfinite().all() for t in got)
    gated_backward_check(got, dh, x, w, pre, act, act)


def test_gated_linear_shapes_strides_and_masks():
    g = generator(21)
    x = randn(g, 130, 3, 2, dtype=torch.bfloat16).permute(2, 1, 0)                # [2, 3, 130], not dense
    w = randn(g, 130, 2 * 40, dtype=torch.bfloat16, scale=0.1).t()                # [80, 130], transposed
    h, pre = ops.gated_linear(x, w, "silu", save_pre=True)
    assert h.shape == (2, 3, 40) and pre.shape == (2, 3, 80)
    xc, wc = x.contiguous().view(6, 130), w.contiguous()
    gated_forward_check(h.view(6, 40), pre.view(6, 80), xc, wc, "silu", "strided")
    dh = randn(g, 40, 3, 2, dtype=torch.bfloat16).permute(2, 1, 0)
    dx, dw = ops.gated_linear_backward(dh, x, w, pre, "silu")
    assert dx.shape == x.shape and dw.shape == w.shape
    dhc = dh.contiguous().view(6, 40)
    gated_backward_check((dx.view(6, 130), dw), dhc, xc, wc, pre.view(6, 80), "silu", "strided")
    one = ops.gated_linear_backward(dh, x, w, pre, "silu", (True, False))
    assert torch.equal(one[0], dx) and one[1] is None
    one = ops.gated_linear_backward(dh, x, w, pre, "silu", (False, True))
    assert one[0] is None and torch.equal(one[1], dw)
    vec = ops.gated_linear(xc[0], wc)                                              # one token without a batch dimension
    assert vec.shape == (40,)
    gated_forward_check(vec.view(1, 40), None, xc[:1], wc, "silu", "vector")
    sliced = randn(g, 9, 300, dtype=torch.float16)[:, 4:260]                       # rows 300 apart, 8 bytes off a boundary
    ws = randn(g, 96, 264, dtype=torch.float16, scale=0.1)[:, :256]
    gated_forward_check(ops.gated_linear(sliced, ws, "gelu"), None, sliced.contiguous(), ws.contiguous(), "gelu", "sliced")
    # overlapping rows: a weight whose rows are all the same storage, tokens that share elements
    same = randn(g, 1, 256, dtype=torch.float16, scale=0.1).expand(64, 256)
    shared = randn(g, 1000, dtype=torch.float16).as_strided((90, 256), (8, 1))
    gated_forward_check(ops.gated_linear(shared, same, "silu"), None, shared.contiguous(), same.contiguous(), "silu", "overlapping")
    dx, dw = ops.gated_linear_backward(shared[:, :32], shared, same, shared[:, :64], "silu")
    gated_backward_check((dx, dw), shared[:, :32].contiguous(), shared.contiguous(), same.contiguous(), shared[:, :64].contiguous(), "silu", "overlapping")


def test_gated_linear_empties():
    for M, K, F in ((0, 16, 8), (4, 0, 8), (4, 16, 0)):
        x, w = torch.ones(M, K, device="cuda"), torch.ones(2 * F, K, device="cuda")
        h, pre = ops.gated_linear(x, w, save_pre=True)
        assert h.shape == (M, F) and pre.shape == (M, 2 * F) and not h.any() and not pre.any()
        dx, dw = ops.gated_linear_backward(torch.ones(M, F, device="cuda"), x, w, pre)
        assert dx.shape == x.shape and dw.shape == w.shape and not dx.any() and not dw.any()


def test_gated_linear_nan_stays_in_its_token():
    for M in (3, 70, 300):
        g = generator(M)
        x, w = randn(g, M, 256, dtype=torch.bfloat16), randn(g, 256, 256, dtype=torch.bfloat16, scale=0.06)
        clean = ops.gated_linear(x, w)
        x[1, 77] = float("nan")
        got = ops.gated_linear(x, w)
        keep = torch.arange(M, device="cuda") != 1
        assert got[1].isnan().all() and torch.equal(got[keep], clean[keep])


# ---- dropout ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,p", [(1, 0.5), (7, 0.5), (8, 0.3), (9, 0.1), (2048, 0.1), (2049, 0.25), (10007, 0.9), (4096, 0.0), (4096, 1.0), (4096, 1e-6)])
def test_dropout_add(n, p, dtype):
    g = generator(n)
    x, r = randn(g, n, dtype=dtype), randn(g, n, dtype=dtype)
    seed, offset = 0x1234567890ABCDEF, 2 ** 32 - 100  # the counter's low word wraps inside the larger ones
    keep = ref.dropout_keep(n, p, seed, offset).cuda()
    drop = torch.where(keep, x.double() * ref.dropout_scale(p), 0.0)
    u = unit(dtype)
    check(ops.dropout_add(x, None, p, (seed, offset)), drop, 2 * u * drop.abs(), "dropout")
    check(ops.dropout_add(x, r, p, (seed, offset)), drop + r.double(), 3 * u * (drop.abs() + r.double().abs()), "dropout + residual")
    state = torch.tensor([seed, offset], device="cuda")
    assert torch.equal(ops.dropout_add(x, r, p, state), ops.dropout_add(x, r, p, (seed, offset)))
    grad = ops.dropout_add_backward(r, p, state)
    assert torch.equal(grad, ops.dropout_add(r, None, p, state))
    assert torch.equal(ops.dropout_add(x, None, p, (seed - 2 ** 64, offset + 2 ** 64)), ops.dropout_add(x, None, p, (seed, offset)))


def test_dropout_offsets_continue():
    """A call over the second part of a tensor with the advanced offset draws what one call over the whole draws."""
    g = generator(31)
    x = randn(g, 4096, dtype=torch.bfloat16)
    whole = ops.dropout_add(x, None, 0.4, (5, 9))
    cut = 1024
    assert ops.dropout_counters(cut) == 128 and ops.dropout_counters(cut + 1) == 129
    rest = ops.dropout_add(x[cut:], None, 0.4, (5, 9 + ops.dropout_counters(cut)))
    assert torch.equal(whole[cut:], rest)
    assert not torch.equal(whole, ops.dropout_add(x, None, 0.4, (6, 9)))
    assert not torch.equal(whole, ops.dropout_add(x, None, 0.4, (5, 9 + 512)))


def test_dropout_strides_alignment_and_dropped_values():
    g = generator(32)
    x, r = randn(g, 60, 70).t(), randn(g, 70, 61)[:, 1:]
    got = ops.dropout_add(x, r, 0.5, (1, 2))
    assert torch.equal(got, ops.dropout_add(x.contiguous(), r.contiguous(), 0.5, (1, 2))) and got.is_contiguous()
    flat = randn(g, 1001, dtype=torch.float16)
    assert torch.equal(ops.dropout_add(flat[1:], None, 0.5, (1, 2)), ops.dropout_add(flat[1:].clone(), None, 0.5, (1, 2)))
    keep = ops.dropout_add(torch.ones(1000, device="cuda"), None, 0.5, (1, 2)) != 0
    bad = torch.where(keep, 1.0, float("nan"))
    assert ops.dropout_add(bad, None, 0.5, (1, 2)).isfinite().all()   # what is dropped is not read into the result
    assert ops.dropout_add(torch.empty(0, 4, device="cuda"), None, 0.5, (1, 2)).shape == (0, 4)
    assert ops.dropout_add(torch.tensor(2.0, device="cuda"), None, 0.0, (1, 2)).item() == 2.0


# ---- devices, streams, graphs ----------------------------------------------------------
def test_cpu_tensors_make_the_round_trip():
    g = torch.Generator().manual_seed(1)
    x, w = torch.randn(6, 64, generator=g), torch.randn(32, 64, generator=g) * 0.1
    h, pre = ops.gated_linear(x, w, save_pre=True)
    assert h.device.type == pre.device.type == "cpu" and torch.equal(h, ops.gated_linear(x.cuda(), w.cuda()).cpu())
    dx, dw = ops.gated_linear_backward(h, x, w, pre, output_mask=(True, False))
    assert dx.device.type == "cpu" and dw is None
    assert torch.equal(ops.dropout_add(x, x, 0.3, (1, 2)), ops.dropout_add(x.cuda(), x.cuda(), 0.3, torch.tensor([1, 2])).cpu())
    s = torch.ones(6, 1)
    dx, dw, db = ops.native_layer_norm_backward(x, x, [64], s, s, torch.ones(64), None, [True, True, False])
    assert dx.device.type == dw.device.type == "cpu" and db is None


class Block:
    """The residual branch of a pre-norm block, forward and backward, on the operators:
    y = x + dropout(gated_linear(layer_norm(x)) @ down^T)."""

    def __init__(self, M, D, F, dtype, seed, p=0.2):
        g = generator(seed)
        self.p, self.D = p, D
        self.x, self.dy = randn(g, M, D, dtype=dtype), randn(g, M, D, dtype=dtype, scale=0.1)
        self.gamma, self.beta = randn(g, D, dtype=dtype, scale=0.1) + 1, randn(g, D, dtype=dtype, scale=0.1)
        self.w, self.down = randn(g, 2 * F, D, dtype=dtype, scale=D ** -0.5), randn(g, D, F, dtype=dtype, scale=F ** -0.5)
        self.rng = torch.tensor([seed, 1000], device="cuda")

    def step(self):
        n, mean, rstd = ops.SLOTS["native_layer_norm__default"](self.x, [self.D], self.gamma, self.beta, 1e-5)
        h, pre = ops.gated_linear(n, self.w, "silu", save_pre=True)
        o = ops.SLOTS["mm__default"](h, self.down.t())
        y = ops.dropout_add(o, self.x, self.p, self.rng)
        do = ops.dropout_add_backward(self.dy, self.p, self.rng)
        ddown = ops.SLOTS["mm__default"](do.t(), h)
        dh = ops.SLOTS["mm__default"](do, self.down)
        dn, dw = ops.gated_linear_backward(dh, n, self.w, pre, "silu")
        dx, dgamma, dbeta = ops.native_layer_norm_backward(dn, self.x, [self.D], mean, rstd, self.gamma, self.beta, [True] * 3)
        return y, ops.SLOTS["add__Tensor"](dx, self.dy), dw, ddown, dgamma, dbeta

    def reference(self):
        M = self.x.shape[0]
        keep = ref.dropout_keep(self.x.numel(), self.p, *self.rng.tolist()).cuda().view(M, self.D)
        leaves = [t.double().requires_grad_() for t in (self.x, self.w, self.down, self.gamma, self.beta)]
        x, w, down, gamma, beta = leaves
        mu = x.mean(1, keepdim=True)
        n = (x - mu) / torch.sqrt((x - mu).square().mean(1, keepdim=True) + 1e-5) * gamma + beta
        pre = n @ w.t()
        F = down.shape[1]
        o = (ref.activation(pre[:, :F], "silu")[0] * pre[:, F:]) @ down.t()
        y = x + torch.where(keep, o * ref.dropout_scale(self.p), 0.0)
        return (y.detach(), *torch.autograd.grad(y, leaves, self.dy.double()))


@pytest.mark.parametrize("M,D,F,dtype", [(67, 256, 344, torch.float32), (300, 512, 688, torch.bfloat16), (1, 128, 96, torch.float16)])
def test_block_together(M, D, F, dtype):
    """Several tensors between the operators are rounded to `dtype`: each adds an independent relative error of at
    most half a step, so the norm of the difference stays under (roundings on the longest path, 10) half steps of the norm;
    fp32's own accumulation (a few hundred roundings) enters as 2^-24 * 512."""
    b = Block(M, D, F, dtype, 41)
    for name, got, want in zip(("y", "dx", "dw", "ddown", "dgamma", "dbeta"), b.step(), b.reference()):
        rel = ((got.double() - want).norm() / want.norm()).item()
        assert rel <= 10 * torch.finfo(dtype).eps / 2 + 512 * 2.0 ** -24, (name, rel)


def test_block_in_a_graph_and_on_another_stream():
    b = Block(150, 256, 344, torch.bfloat16, 43)
    eager = [t.clone() for t in b.step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = b.step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, c) for a, c in zip(eager, other))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = b.step()
    for step in range(4):
        b.rng[1] = 1000 + 7 * step
        b.x.copy_(randn(generator(step), 150, 256, dtype=torch.bfloat16))
        graph.replay()
        replayed = [t.clone() for t in out]
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(replayed, b.step())), step
    assert _lib.load().mi355_gemm_status() == 0
