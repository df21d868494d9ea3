"""Definitions of the int8 operators and how far a kernel may be off them.

quantize: the three fp32 operations of the definition, so that whole numbers and
scales are compared exactly.  linear: 64 bits from the int8 operands; the kernel
rounds the exact sum to fp32, multiplies it by two scales and adds the bias, four
roundings of 2^-24 each, then goes on as the 16-bit layers do (layer_refs.py).
"""
import torch

import layer_refs as R


def quantize(x):
    """(q, scale) of x's rows, by fp32 operations."""
    x = x.float()
    top = x.abs().amax(1) if x.shape[1] else torch.zeros(x.shape[0], device=x.device)
    top = torch.where(top < 2.0 ** -100, torch.full_like(top, 2.0 ** -100), top)  # NaN stays
    finite = torch.isfinite(top)
    # IEEE quotients through 64 bits (rounding twice is harmless there): torch divides by and into Python numbers by way
    # of rounded reciprocals
    r, scale = (127.0 / top.double()).float(), (top.double() / 127.0).float()
    q = torch.round(torch.where(finite[:, None], x, torch.zeros_like(x)) * r[:, None])
    return torch.where(finite[:, None], q, torch.zeros_like(q)).to(torch.int8), scale


def linear(xq, xs, wq, ws, bias, residual, act, dt, gated):
    """(y, bound) in 64 bits."""
    z = (xq.double() @ wq.double().t()) * xs.double()[:, None] * ws.double()
    ez = 3 * 2.0 ** -24 * z.abs()
    if bias is not None:
        z = z + bias.double()
        ez = ez + 2.0 ** -24 * z.abs()
    ez = 1.001 * ez  # products of the errors
    n = wq.shape[0] // 2 if gated else wq.shape[0]
    a, ea = z[:, :n], ez[:, :n]
    v = R.value(a, act)
    ev = R.SLOPE[act] * ea + R.act_error(a, act) * (v.abs() + ea) + R.act_floor(a, act)
    y, ey = v, ev
    if gated:
        b, eb = z[:, n:], ez[:, n:]
        y = v * b
        ey = ev * b.abs() + v.abs() * eb + ev * eb + 2.0 ** -23 * y.abs()
    if residual is not None:
        y = y + residual.double()
        ey = ey + 2.0 ** -23 * (y.abs() + ey)
    return y, R.u(dt) * y.abs() + (1 + R.u(dt)) * ey + R.TINY[dt]
