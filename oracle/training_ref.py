"""float64 restatements of the training operators' definitions, in torch on the inputs' device (test infrastructure,
see oracle/__init__.py).  Each returns the value and, beside it, what the rounding errors of an fp32 kernel are
measured against: the same sum with every term's absolute value."""

import math

import torch


def layer_norm_backward(dy, x, mean, rstd, weight, rows, cols):
    """((dx, dw, db), (scales)) over `rows` x `cols`; weight None: ones."""
    dy, x = dy.double().reshape(rows, cols), x.double().reshape(rows, cols)
    mean, rstd = mean.double().reshape(rows, 1), rstd.double().reshape(rows, 1)
    w = weight.double().reshape(1, cols) if weight is not None else torch.ones(1, cols, dtype=torch.float64, device=x.device)
    xhat = (x - mean) * rstd
    g = dy * w
    m1, m2 = g.mean(1, keepdim=True), (g * xhat).mean(1, keepdim=True)
    dx = rstd * (g - m1 - xhat * m2)
    sx = rstd * (g.abs() + g.abs().mean(1, keepdim=True) + xhat.abs() * (g * xhat).abs().mean(1, keepdim=True))
    return (dx, (dy * xhat).sum(0), dy.sum(0)), (sx, (dy * xhat).abs().sum(0), dy.abs().sum(0))


def activation(g, name):
    """(act(g), act'(g))"""
    if name == "silu":
        s = torch.sigmoid(g)
        return g * s, s + g * s * (1 - s)
    if name == "gelu":
        phi = 0.5 * torch.erfc(-g * math.sqrt(0.5))
        return g * phi, phi + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
    c = math.sqrt(2 / math.pi)
    s = torch.sigmoid(2 * c * (g + 0.044715 * g ** 3))
    return g * s, s + g * 2 * s * (1 - s) * c * (1 + 3 * 0.044715 * g * g)


def gated_linear(x, weight, name):
    """((h, pre), pre's scale): x [M, K], weight [2F, K]."""
    x, weight = x.double(), weight.double()
    pre = x @ weight.t().contiguous()
    F = weight.shape[0] // 2
    return (activation(pre[:, :F], name)[0] * pre[:, F:], pre), x.abs() @ weight.abs().t().contiguous()


def gated_pre_backward(dh, pre, name):
    """d pre [M, 2F]"""
    F = pre.shape[1] // 2
    dh, g, u = dh.double(), pre[:, :F].double(), pre[:, F:].double()
    a, da = activation(g, name)
    return torch.cat([dh * u * da, dh * a], 1)


def philox4x32_10(counter, key):
    """The four 32-bit outputs of Philox-4x32-10 (Salmon, Moraes, Dror, Shaw, 2011), Python integers."""
    c, k = list(counter), list(key)
    for _ in range(10):
        p0, p1 = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(p1 >> 32) ^ c[1] ^ k[0], p1 & 0xFFFFFFFF, (p0 >> 32) ^ c[3] ^ k[1], p0 & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def dropout_keep(n, p, seed, offset):
    """bool [n] on the CPU: which elements dropout keeps."""
    t = round(p * 65536)  # halves to even
    draws = []
    for i in range((n + 7) // 8):
        ctr = (offset + i) % 2 ** 64
        seed %= 2 ** 64
        for word in philox4x32_10((ctr & 0xFFFFFFFF, ctr >> 32, 0, 0), (seed & 0xFFFFFFFF, seed >> 32)):
            draws += [word & 0xFFFF, word >> 16]
    return torch.tensor([d >= t for d in draws[:n]], dtype=torch.bool)


def dropout_scale(p):
    t = round(p * 65536)  # halves to even
    return 65536.0 / (65536 - t) if t < 65536 else 0.0
