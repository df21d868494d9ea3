"""64-bit definitions of the feed-forward layer operators and how far a kernel
may be off them, element by element.

Every bound counts roundings.  u(t) = eps(t) / 2 is the largest relative error
of one rounding to type t; TINY(t) is half the spacing of its smallest values.
A sum of K products in fp32, in any order and with each addition off by at most
2^-23 of its result (tensor cores cut low bits off instead of rounding), is off
by at most (K + 8) 2^-23 times the sum of the products' absolute values.
"""
import math

import torch

ACTS = ("none", "relu", "gelu", "gelu_tanh", "silu", "sigmoid")
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}
# Largest |act'| and |act''| over the reals, rounded up (relu's second
# derivative is left out: the tests keep z away from 0 where it would matter).
SLOPE = {"none": 1.0, "relu": 1.0, "gelu": 1.13, "gelu_tanh": 1.13, "silu": 1.1, "sigmoid": 0.25}
CURVE = {"none": 0.0, "relu": 0.0, "gelu": 0.8, "gelu_tanh": 0.81, "silu": 0.5, "sigmoid": 0.1}


def u(dtype):
    return torch.finfo(dtype).eps / 2


def value(z, act):
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "gelu":
        return z * 0.5 * torch.special.erfc(-z / math.sqrt(2))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "sigmoid":
        return torch.sigmoid(z)
    return z


def slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        return 0.5 * torch.special.erfc(-z / math.sqrt(2)) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z ** 3))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 0.134145 * z * z)
    if act == "silu":
        s = torch.sigmoid(z)
        return s + z * s * (1 - s)
    if act == "sigmoid":
        s = torch.sigmoid(z)
        return s * (1 - s)
    return torch.ones_like(z)


def act_floor(z, act):
    """Absolute error of act (and of act') at z beside act_error: gelu's distribution function comes from a published
    rational form (Abramowitz and Stegun, 26.2.17) whose error is below 7.5e-8; 1 - q adds one rounding, 2^-25."""
    return 1.05e-7 * (z.abs() + 1) if act == "gelu" else torch.zeros_like(z)


def act_error(z, act):
    """Relative error of one fp32 evaluation of act (or of act' beside it) at z.
    exp(t) is off by 2 units in the last place plus |t| 2^-24 from rounding its
    argument; the argument itself, with up to four roundings, by 4 |t| 2^-24."""
    if act in ("none", "relu"):
        return torch.zeros_like(z)
    if act == "gelu":  # exp(-z^2 / 2)
        t = z * z / 2
    elif act == "gelu_tanh":
        t = (1.6 * (z + 0.044715 * z ** 3)).abs()
    else:
        t = z.abs()
    return (5 * t + 32) * 2.0 ** -24


def linear(x, w, bias, residual, act, trans_w, gated):
    """(y, z, bound of y, bound of z) in 64 bits."""
    dt = x.dtype
    X, W = x.double(), (w.t() if trans_w else w).double()
    z = X @ W
    size = X.abs() @ W.abs()
    if bias is not None:
        z = z + bias.double()
        size = size + bias.double().abs()
    ez = (X.shape[1] + 8) * 2.0 ** -23 * size
    n = W.shape[1] // 2 if gated else W.shape[1]
    a, ea = z[:, :n], ez[:, :n]
    v = value(a, act)
    # sigmoid and its relatives: near 0 the relative error counts, so bound the value's own change
    ev = SLOPE[act] * ea + act_error(a, act) * (v.abs() + ea) + act_floor(a, act)
    y, ey = v, ev
    if gated:
        b, eb = z[:, n:], ez[:, n:]
        y = v * b
        ey = ev * b.abs() + v.abs() * eb + ev * eb + 2.0 ** -23 * y.abs()
    if residual is not None:
        y = y + residual.double()
        ey = ey + 2.0 ** -23 * (y.abs() + ey)
    return y, z, u(dt) * y.abs() + (1 + u(dt)) * ey + TINY[dt], u(dt) * z.abs() + (1 + u(dt)) * ez + TINY[dt]


def linear_backward(dy, x, w, z, act, trans_w, gated):
    """((dx, bound), (dw, bound), (db, bound)) in 64 bits for a stored z."""
    dt = dy.dtype
    g, X, W = dy.double(), x.double(), (w.t() if trans_w else w).double()
    m, n = g.shape
    if gated:
        a, b = z[:, :n].double(), z[:, n:].double()
        d = torch.cat((g * b * slope(a, act), g * value(a, act)), 1)
        # act' is a sum of two terms, each at most 1.2 in size and evaluated to act_error
        f = act_floor(a, act)
        e = torch.cat(((g * b).abs() * (3 * act_error(a, act) + 2.0 ** -22 + f),
                       d[:, n:].abs() * (act_error(a, act) + 2.0 ** -23) + g.abs() * f), 1)
    elif act == "none":
        d, e = g, torch.zeros_like(g)
    else:
        d = g * slope(z.double(), act)
        e = g.abs() * (3 * act_error(z.double(), act) + 2.0 ** -22 + act_floor(z.double(), act))
    rounded = e if (act == "none" and not gated) else e + u(dt) * (d.abs() + e) + TINY[dt]

    def product(A, eA, B):
        size = A.abs() @ B.abs() + eA @ B.abs()
        p = A @ B
        return p, u(dt) * p.abs() + (1 + u(dt)) * (eA @ B.abs() + (A.shape[1] + 8) * 2.0 ** -23 * size) + TINY[dt]

    dx = product(d, rounded, W.t())
    dw = product(d.t(), rounded.t(), X)  # [wide][K]
    if not trans_w:
        dw = (dw[0].t(), dw[1].t())
    db = d.sum(0)
    edb = e.sum(0) + (m + 8) * 2.0 ** -23 * (d.abs() + e).sum(0)
    return dx, dw, (db, u(dt) * db.abs() + (1 + u(dt)) * edb + TINY[dt])


def layer_norm(x, weight, bias, eps):
    """(y, mean, rstd, bound of y, of mean, of rstd) in 64 bits."""
    dt = x.dtype
    X = x.double()
    n = X.shape[1]
    mean = X.mean(1)
    d = X - mean[:, None]
    var = (d * d).mean(1)
    rstd = (var + eps) ** -0.5
    h = d * rstd[:, None]
    q = (n + 8) * 2.0 ** -24
    emean = q * X.abs().mean(1) + 2.0 ** -24 * mean.abs()
    # d is off by the mean's error and one rounding; var by what that gives and its own sum
    ed = emean[:, None] + 2.0 ** -24 * d.abs()
    evar = (2 * d.abs() * ed + ed * ed).mean(1) + (q + 2.0 ** -23) * var
    # relative error of rstd: half of (var + eps)'s, to first order; doubled for the rest
    rel = evar / (var + eps) + 3 * 2.0 ** -23
    w = torch.ones(n, dtype=torch.float64, device=x.device) if weight is None else weight.double()
    b = torch.zeros(n, dtype=torch.float64, device=x.device) if bias is None else bias.double()
    y = h * w + b
    ey = (ed * rstd[:, None] + h.abs() * (rel[:, None] + 2.0 ** -22)) * w.abs() * (1 + rel[:, None]) + 2.0 ** -23 * y.abs()
    return y, mean, rstd, u(dt) * y.abs() + (1 + u(dt)) * ey + TINY[dt], emean, rel * rstd


def layer_norm_backward(dy, x, mean, rstd, weight):
    """((dx, bound), (dw, bound), (db, bound)) in 64 bits for the given fp32 statistics."""
    dt = x.dtype
    wt = dt if weight is None else weight.dtype
    m, n = x.shape
    r = rstd.double()[:, None]
    h = (x.double() - mean.double()[:, None]) * r
    eh = 2.0 ** -23 * h.abs()
    g = dy.double()
    t = g if weight is None else g * weight.double()
    et = 2.0 ** -24 * t.abs()
    q = (n + 8) * 2.0 ** -24
    a0, a1 = t.mean(1, keepdim=True), (t * h).mean(1, keepdim=True)
    e0 = (et + q * t.abs()).mean(1, keepdim=True) + 2.0 ** -23 * a0.abs()
    e1 = ((t * h).abs() * (q + 2.0 ** -22)).mean(1, keepdim=True) + 2.0 ** -23 * a1.abs()
    dx = r * (t - a0 - h * a1)
    edx = r * (et + e0 + eh * a1.abs() + h.abs() * e1 + 2.0 ** -22 * (t.abs() + a0.abs() + (h * a1).abs()))
    s = (m + 8) * 2.0 ** -24
    dw, db = (g * h).sum(0), g.sum(0)
    edw = ((g * h).abs() * (s + 2.0 ** -22)).sum(0)
    edb = (g.abs() * s).sum(0)

    def out(v, e, t):
        return v, u(t) * v.abs() + (1 + u(t)) * e + TINY[t]

    return out(dx, edx, dt), out(dw, edw, wt), out(db, edb, wt)


def philox_words(count, seed, offset):
    """The dropout generator in Python integers (Philox4x32-10, Salmon et al. 2011)."""
    words = []
    for g in range((count + 3) // 4):
        ctr = (offset + g) % 2 ** 64
        c = [ctr % 2 ** 32, ctr >> 32, 0, 0]
        k0, k1 = seed % 2 ** 32, (seed >> 32) % 2 ** 32
        for _ in range(10):
            p0, p1 = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
            c = [(p1 >> 32) ^ c[1] ^ k0, p1 % 2 ** 32, (p0 >> 32) ^ c[3] ^ k1, p0 % 2 ** 32]
            k0, k1 = (k0 + 0x9E3779B9) % 2 ** 32, (k1 + 0xBB67AE85) % 2 ** 32
        words += c
    return words[:count]


def assert_within(got, ref, bound, what=""):
    got = got.double()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    bad = ~((got - ref).abs() <= bound)
    if bad.any():
        i = tuple(bad.nonzero()[0].tolist())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {i}: {got[i].item()!r} for "
                             f"{ref[i].item()!r}, allowed {bound[i].item():.3g}")
