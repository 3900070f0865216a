"""Calls of the training operators that the documentation allows beside the ordinary ones, on the GPU, against the float64
definitions with the tolerances of tests/test_training_gpu.py."""

import threading

import pytest
import torch

from backendbench_amd import _lib, ops
from backendbench_amd.ops import elementwise, training
from oracle import training_ref as ref
from test_training_gpu import DTYPES, HALF, check, gated_backward_check, gated_forward_check, generator, ln_case, ln_check, randn, unit

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


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("K,F", [(1, 9), (16, 40), (17, 33), (2048, 24)])
def test_gated_linear_one_row_of_any_stride(K, F, dtype):
    """One token whose row stride torch reports as 1, 0 or an odd distance: the result of the dense row."""
    g = generator(K + F)
    w = randn(g, 2 * F, K, dtype=dtype, scale=K ** -0.5)
    column = randn(g, K, 1, dtype=dtype)
    dense = column.t().clone(memory_format=torch.contiguous_format).view(1, K)
    h, pre = ops.gated_linear(dense, w, "gelu", save_pre=True)
    gated_forward_check(h, pre, dense, w, "gelu", "dense")
    dh = randn(g, 1, F, dtype=dtype)
    grads = ops.gated_linear_backward(dh, dense, w, pre, "gelu")
    gated_backward_check(grads, dh, dense, w, pre, "gelu", "dense")
    far = torch.full((3, K + 5), float("nan"), device="cuda", dtype=dtype)[1:2, :K]
    far.copy_(dense)
    got, gpre = ops.gated_linear(far, w, "gelu", save_pre=True)  # (another address, so perhaps another kernel)
    gated_forward_check(got, gpre, dense, w, "gelu", "far")
    gated_backward_check(ops.gated_linear_backward(dh, far, w, pre, "gelu"), dh, dense, w, pre, "gelu", "far")
    for x in (column.t(), dense[0].expand(4, K)[:1], dense.as_strided((1, K), (0, 1)), dense.view(1, 1, K).as_strided((1, 1, K), (1, 1, 1))):
        got, gpre = ops.gated_linear(x, w, "gelu", save_pre=True)
        assert torch.equal(got.view(1, F), h) and torch.equal(gpre.view(1, 2 * F), pre)
        back = ops.gated_linear_backward(dh.view_as(got), x, w, gpre, "gelu")
        assert torch.equal(back[0].view(1, K), grads[0]) and torch.equal(back[1], grads[1])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("halves", [1, 3, 5, 7, 65535, 131071])
def test_dropout_probabilities_halfway_between_two_steps(halves, dtype):
    """p in the middle of two 65536ths goes to the even one; 2^-17 is no dropout at all."""
    p, n = halves * 2.0 ** -17, 5003
    x = randn(generator(halves), n, dtype=dtype)
    keep = ref.dropout_keep(n, p, 77, 5).cuda()
    want = torch.where(keep, x.double() * ref.dropout_scale(p), 0.0)
    got = ops.dropout_add(x, None, p, (77, 5))
    check(got, want, 2 * unit(dtype) * want.abs(), f"p = {halves} / 2^17")
    if halves == 1:
        assert torch.equal(got, x)


@pytest.mark.parametrize("x_more,w_more", [(0, 1), (1, 0), (3, 2), (4, 8)])
def test_gated_linear_f32_rows_off_16_bytes_go_through_padded_copies(monkeypatch, x_more, w_more):
    """fp32, more rows than the fused kernels take: rows that do not start on 16-byte boundaries are padded like an odd K."""
    M, K, F = 70, 256, 72
    g = generator(61)
    x, w = randn(g, M, K + x_more), randn(g, 2 * F, K + w_more, scale=K ** -0.5)
    x[:, K:], w[:, K:] = float("nan"), float("nan")
    calls, padded = [], training._padded
    monkeypatch.setattr(training, "_padded", lambda t, columns: calls.append(columns) or padded(t, columns))
    h, pre = ops.gated_linear(x[:, :K], w[:, :K], "silu", save_pre=True)
    gated_forward_check(h, pre, x[:, :K].contiguous(), w[:, :K].contiguous(), "silu", f"{x_more} {w_more}")
    assert calls == ([] if x_more % 4 == 0 and w_more % 4 == 0 else [K, K])


@pytest.mark.parametrize("M,K,F", [(33, 512, 4096), (64, 512, 4160), (64, 2176, 4160), (33, 2176, 8192), (40, 2048, 4104), (64, 2112, 8256)])
def test_gated_linear_on_both_sides_of_the_rule_for_33_to_64_rows(M, K, F):
    """One round of the CUs for the rows' kernel, two, and more; short and long K."""
    g = generator(M + K + F)
    x, w = randn(g, M, K, dtype=torch.bfloat16), randn(g, 2 * F, K, dtype=torch.bfloat16, scale=K ** -0.5)
    h, pre = ops.gated_linear(x, w, "silu", save_pre=True)
    gated_forward_check(h, pre, x, w, "silu", f"{M}x{K}x{F}")
    assert torch.equal(ops.gated_linear(x, w, "silu"), h)


def inside(t, before, after, rows=1):
    """`t` [R, C] as a view of a wider, taller tensor of NaN."""
    wide = torch.full((t.shape[0] + rows, t.shape[1] + before + after), float("nan"), device="cuda", dtype=t.dtype)
    view = wide[:t.shape[0], before:before + t.shape[1]]
    view.copy_(t)
    return view


# Many features (blocks of 16 of them), aligned rows with whole chunks and a rest behind them, and odd ones; every count of rows
# that picks another ring.
@pytest.mark.parametrize("M", [3, 5, 16, 17, 32, 33, 64])
@pytest.mark.parametrize("K,F", [(1016, 2056), (4104, 2056), (264, 4099), (777, 4099), (4099, 2056)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_gated_linear_few_rows_many_features(dtype, K, F, M):
    g = generator(M + K + F)
    x, w = randn(g, M, K, dtype=dtype), randn(g, 2 * F, K, dtype=dtype, scale=K ** -0.5)
    around = (8, 16) if K % 8 == 0 else (3, 2)
    act = ["silu", "gelu", "gelu_tanh"][M % 3]
    h, pre = ops.gated_linear(inside(x, *around), inside(w, *around), act, save_pre=True)
    gated_forward_check(h, pre, x, w, act, f"{M}x{K}x{F} {act}")
    assert torch.equal(ops.gated_linear(inside(x, *around), inside(w, *around), act), h)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K,F", [(4, 4096, 4099), (8, 4100, 2051), (16, 2049, 4099), (12, 1032, 4200), (3, 8200, 1100)])
def test_gated_linear_backward_few_rows_several_steps(dtype, M, K, F):
    """A group of features takes several steps, over which the sums of dx are carried; each gradient alone gives the same."""
    g = generator(M + K + F)
    x, w = randn(g, M, K, dtype=dtype), randn(g, 2 * F, K, dtype=dtype, scale=K ** -0.5)
    pre, dh = randn(g, M, 2 * F, dtype=dtype), randn(g, M, F, dtype=dtype)
    act = ["silu", "gelu", "gelu_tanh"][F % 3]
    xv, wv = inside(x, 1, 4), inside(w, 3, 2)
    got = ops.gated_linear_backward(dh, xv, wv, pre, act)
    gated_backward_check(got, dh, x, w, pre, act, f"{M}x{K}x{F} {act}")
    dx, none = ops.gated_linear_backward(dh, xv, wv, pre, act, (True, False))
    assert none is None and torch.equal(dx, got[0])
    none, dw = ops.gated_linear_backward(dh, xv, wv, pre, act, (False, True))
    assert none is None and torch.equal(dw, got[1])


@pytest.mark.parametrize("rows,cols", [(300, 16384), (261, 16381), (600, 8200), (1030, 8193), (259, 12003)])
@pytest.mark.parametrize("dtype,wdtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32),
                                          (torch.float16, torch.float16), (torch.float16, torch.float32)])
def test_layer_norm_backward_long_rows_on_many_blocks(dtype, wdtype, rows, cols):
    """Rows of 8 K - 16 K elements, a row per block at a time: several blocks with several rows each, their partial sums
    and the pass that adds those."""
    case = ln_case(rows, cols, dtype, wdtype, rows + cols)
    got = ops.native_layer_norm_backward(case[0], case[1], [cols], *case[2:], [True] * 3)
    ln_check(got, *case[:5], rows, cols, f"[{rows}, {cols}]")
    none, dw, db = ops.native_layer_norm_backward(case[0], case[1], [cols], *case[2:], [False, True, True])
    assert none is None and torch.equal(dw, got[1]) and torch.equal(db, got[2])


@pytest.fixture
def gated_form():
    yield lambda value: _lib.set_knob("gated_form", value)
    _lib.set_knob("gated_form", None)


@pytest.mark.parametrize("off", [0, 1])
@pytest.mark.parametrize("form,M,K,F", [
    ("dots", 2, 1331, 33), ("rows", 3, 1016, 24), ("rows", 16, 777, 2061), ("rows", 33, 520, 70), ("rows", 64, 512, 64),
    ("tile128", 1, 64, 1), ("tile128", 130, 192, 70), ("tile128", 257, 448, 200), ("tile128", 128, 1024, 64),
    ("tile256", 1, 256, 1), ("tile256", 300, 384, 129), ("tile256", 257, 640, 136), ("tile256", 512, 256, 256)])
@pytest.mark.parametrize("dtype", HALF)
def test_gated_linear_reads_and_writes_its_operands_alone(gated_form, form, M, K, F, off, dtype):
    """Every kernel form with NaN around x and the weight and marks around h and pre, the results on and off a 16-byte boundary."""
    g = generator(M + K + F)
    x, w = randn(g, M, K, dtype=dtype), randn(g, 2 * F, K, dtype=dtype, scale=K ** -0.5)
    around = (3, 2) if K % 8 else (8, 16)
    xv, wv = inside(x, *around), inside(w, *around)
    mark, edge = 7.0, 4096
    out = [torch.full((edge + off + M * n + edge,), mark, device="cuda", dtype=dtype) for n in (F, 2 * F)]
    h, pre = (o[edge + off:edge + off + M * n] for o, n in zip(out, (F, 2 * F)))
    gated_form(form)
    rc = _lib.load().mi355_gated_linear(xv.data_ptr(), xv.stride(0), wv.data_ptr(), wv.stride(0), h.data_ptr(), pre.data_ptr(), M, F, K,
                                        _lib.GELU, _lib.DTYPE[dtype], _lib.current_stream_handle())
    assert rc == 0
    gated_forward_check(h.view(M, F), pre.view(M, 2 * F), x, w, "gelu", f"{form} {M}x{K}x{F}")
    for o, r in zip(out, (h, pre)):
        assert (o[:edge + off] == mark).all() and (o[edge + off + r.numel():] == mark).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K,F", [(1, 8, 3), (5, 77, 33), (16, 1032, 200), (17, 40, 33), (64, 256, 64), (130, 77, 50), (257, 640, 136)])
def test_gated_linear_backward_reads_and_writes_its_operands_alone(M, K, F, dtype):
    """NaN around x and the weight, marks around dx, dweight and the workspace, which holds NaN before the call."""
    g = generator(M + K + F)
    x, w = randn(g, M, K, dtype=dtype), randn(g, 2 * F, K, dtype=dtype, scale=K ** -0.5)
    pre, dh = randn(g, M, 2 * F, dtype=dtype), randn(g, M, F, dtype=dtype)
    xv, wv = inside(x, 3, 2), inside(w, 8, 16)
    lib, code, mark, edge = _lib.load(), _lib.DTYPE[dtype], 7.0, 4096
    out = [torch.full((2 * edge + n * K,), mark, device="cuda", dtype=dtype) for n in (M, 2 * F)]
    dx, dw = (o[edge:edge + n * K] for o, n in zip(out, (M, 2 * F)))
    need = lib.mi355_gated_linear_backward_workspace_bytes(M, F, K, code)
    ws = torch.full((need + 2 * edge,), 255, device="cuda", dtype=torch.uint8)
    rc = lib.mi355_gated_linear_backward(dh.data_ptr(), xv.data_ptr(), xv.stride(0), wv.data_ptr(), wv.stride(0), pre.data_ptr(), dx.data_ptr(),
                                         dw.data_ptr(), M, F, K, _lib.GELU, code, ws.data_ptr() + edge, need, _lib.current_stream_handle())
    assert rc == 0
    gated_backward_check((dx.view(M, K), dw.view(2 * F, K)), dh, x, w, pre, "gelu", f"{M}x{K}x{F}")
    for o, r in zip(out, (dx, dw)):
        assert (o[:edge] == mark).all() and (o[edge + r.numel():] == mark).all()
    assert (ws[:edge] == 255).all() and (ws[edge + need:] == 255).all()


@pytest.mark.parametrize("off", [0, 1])
@pytest.mark.parametrize("rows,cols", [(2, 5), (700, 24), (300, 136), (9, 1001), (517, 4096), (258, 9001), (5, 16500)])
@pytest.mark.parametrize("dtype,wdtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.float16, torch.float16),
                                          (torch.float64, torch.float64)])
def test_layer_norm_backward_writes_its_results_alone(dtype, wdtype, rows, cols, off):
    """Marks around the three gradients and the workspace, which holds NaN before the call; results on and off a 16-byte boundary."""
    dy, x, mean, rstd, w, b = ln_case(rows, cols, dtype, wdtype, rows + cols)
    lib, mark, edge = _lib.load(), 7.0, 4096
    out = [torch.full((2 * edge + off + n,), mark, device="cuda", dtype=d) for n, d in ((rows * cols, dtype), (cols, wdtype), (cols, wdtype))]
    got = [o[edge + off:o.numel() - edge] for o in out]
    need = lib.mi355_layer_norm_backward_workspace_bytes(rows, cols, _lib.DTYPE[dtype])
    ws = torch.full((need + 2 * edge,), 255, device="cuda", dtype=torch.uint8)
    rc = lib.mi355_layer_norm_backward(dy.data_ptr(), x.data_ptr(), _lib.DTYPE[dtype], mean.data_ptr(), rstd.data_ptr(), w.data_ptr(),
                                       _lib.DTYPE[wdtype], *(t.data_ptr() for t in got), rows, cols, ws.data_ptr() + edge, need,
                                       _lib.current_stream_handle())
    assert rc == 0
    ln_check(got, dy, x, mean, rstd, w, rows, cols, f"[{rows}, {cols}]")
    for o in out:
        assert (o[:edge + off] == mark).all() and (o[o.numel() - edge:] == mark).all()
    assert (ws[:edge] == 255).all() and (ws[edge + need:] == 255).all()


def test_operators_on_two_threads_at_once():
    """Each thread on a stream of its own, a hundred rounds of every operator: the bits of a thread alone."""
    def work(seed):
        g = generator(seed)
        dt = torch.bfloat16
        x, w = randn(g, 40, 512, dtype=dt), randn(g, 2 * 344, 512, dtype=dt, scale=0.05)
        dh = randn(g, 40, 344, dtype=dt)
        mean, rstd, gamma = torch.zeros(40, 1, device="cuda"), torch.ones(40, 1, device="cuda"), randn(g, 512, dtype=dt)
        odd, odd_w = randn(g, 70, 301), randn(g, 2 * 33, 301)

        def step():
            h, pre = ops.gated_linear(x, w, "silu", save_pre=True)
            return (h, *ops.gated_linear_backward(dh, x, w, pre, "silu"), ops.dropout_add(x, x, 0.3, (seed, 5)), ops.gated_linear(odd, odd_w, "gelu"),
                    *ops.native_layer_norm_backward(x, x, [512], mean, rstd, gamma, gamma, [True] * 3))
        return step

    steps = [work(71), work(72)]
    alone = [[t.clone() for t in s()] for s in steps]
    torch.cuda.synchronize()
    start, wrong, ended = threading.Barrier(2), [], []

    def thread(i):
        start.wait(60)
        with torch.cuda.stream(torch.cuda.Stream()):
            for n in range(100):
                if not all(torch.equal(a, b) for a, b in zip(alone[i], steps[i]())):
                    wrong.append((i, n))
        ended.append(i)

    threads = [threading.Thread(target=thread, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert sorted(ended) == [0, 1] and not wrong


@pytest.mark.parametrize("M", [5, 16, 40, 300])
def test_gated_linear_backward_f16_overflow_stays_in_its_row(M):
    """f16: a gradient of pre beyond 65504 is infinite in its row of grad_input and its row of grad_weight and reaches nothing else."""
    K, F, m0, f0 = 264, 136, 3, 77
    g = generator(M)
    x, w = randn(g, M, K, dtype=torch.float16), randn(g, 2 * F, K, dtype=torch.float16, scale=0.06)
    pre, dh = randn(g, M, 2 * F, dtype=torch.float16), randn(g, M, F, dtype=torch.float16)
    clean = ops.gated_linear_backward(dh, x, w, pre)
    dh[m0, f0], pre[m0, f0], pre[m0, F + f0] = 60000.0, 3.0, 50.0  # d gate 3.3e6, d up 1.7e5
    dx, dw = ops.gated_linear_backward(dh, x, w, pre)
    rows, features = torch.ones(M, dtype=torch.bool, device="cuda"), torch.ones(2 * F, dtype=torch.bool, device="cuda")
    rows[m0], features[f0], features[F + f0] = False, False, False
    assert torch.equal(dx[rows], clean[0][rows]) and torch.equal(dw[features], clean[1][features])
    assert not dx[m0].isfinite().any() and not dw[~features].isfinite().any()
