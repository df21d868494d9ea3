"""8-bit integer layers for torch tensors over the C ABI: a linear layer's weights and
activations as int8, with one scale for each output column and each row, for serving.

  quantize_int8(x, ...)            q = rint(x * (127 / a)), scale = a / 127, a each row's largest magnitude
  int8_linear(x, w, w_scale, ...)  y = act(x_scale w_scale (xq wq^T) + bias) + residual
  int8_gated_linear(x, w, ...)     y = act(g) * u, [g | u] = x_scale w_scale (xq wq^T) + bias

Calls run on their tensors' device and on `stream`, as in layers.py; there are no gradients.
"""
from __future__ import annotations

from struct import Struct
from typing import Optional

import torch

from . import _native as N
from .layers import _DT, _DT16, _activation, _current_device, _device, _elsewhere, _error, _matrix, _raw_stream, _vector

# The argument structs of include/cuopx.h.
_QUANTIZE = Struct("=2i2qQqQqQQQ")
_INT8 = Struct("=2i3qQqQQqQQQqQqQQ")

_empty = torch.empty


def quantize_int8(x: torch.Tensor, *, trans: bool = False, out: Optional[torch.Tensor] = None,
                  scale: Optional[torch.Tensor] = None, stream=None):
    """(q, scale) of a matrix x, float32, float16 or bfloat16 (cuopx_quantize).

    Without trans each row has a scale (activations: each token; weights stored
    [N, K]); with trans each column of x [K, N] has one and q is [N, K], the
    layout in which int8_linear takes weights.  q's rows start on 16-byte
    boundaries unless `out` says otherwise; a row's largest magnitude counts as
    2^-100 at least, and a row with an infinity or a NaN gets that as its scale
    and zeros.  x is about q * scale, half a step off at most."""
    dtype = x.dtype
    code = _DT.get(dtype)
    device = _device(x, "quantize_int8")
    if code is None:
        _error(N.UNSUPPORTED_TYPE, f"quantize_int8: {dtype}")
    if stream is not None or device != _current_device():
        return _elsewhere(quantize_int8, device, stream, x, trans=trans, out=out, scale=scale)
    if x.dim() != 2:
        _error(N.SHAPE_MISMATCH, "quantize_int8: x must be a matrix")
    rows, cols = x.shape
    ldx = _matrix(x, rows, cols, dtype, device, "x")
    m, k = (cols, rows) if trans else (rows, cols)
    if out is None:
        ldq = (k + 15) & ~15
        out = _empty((m, ldq), dtype=torch.int8, device=x.device)
        if ldq != k:
            out = out[:, :k]
    else:
        ldq = _matrix(out, m, k, torch.int8, device, "out")
    if scale is None:
        scale = _empty(m, dtype=torch.float32, device=x.device)
    sp = _vector(scale, m, torch.float32, device, "scale")
    head = (code, 1 if trans else 0, rows, cols, x.data_ptr(), ldx, out.data_ptr(), ldq, sp)
    lib = N.lib()
    ws = None
    wsb = lib.cuopx_quantize_workspace_size(_QUANTIZE.pack(*head, 0, 0)) if trans else 0
    if wsb:
        ws = _empty(wsb, dtype=torch.uint8, device=x.device)
    rc = lib.cuopx_quantize(_QUANTIZE.pack(*head, ws.data_ptr() if wsb else 0, wsb), _raw_stream(device))
    if rc:
        N.check(rc, "cuopx_quantize")
    return out, scale


def _scratch(size, head) -> int:
    """What the size call says for these arguments, without the call (0.6 us of a 17 us step) where nothing is copied
    and the product's kernel does not quantise x: nothing for an int8 x, else the quantised x and its scales."""
    _, _, m, n, k, xp, ldx, xsp, wp, ldw = head[:10]
    if (wp | ldw) & 15 or (xsp and (xp | ldx) & 15):
        return size(_INT8.pack(*head, 0, 0))
    if xsp or not (m and n and k):
        return 0
    if m * k <= 8192:  # the product's kernel may quantise x
        return size(_INT8.pack(*head, 0, 0))
    return ((m * ((k + 15) & ~15) + 255) & ~255) + ((4 * m + 255) & ~255)


def _int8(fn, gated: bool, x, w, w_scale, bias, residual, x_scale, activation, dtype, out, stream):
    what = "int8_gated_linear" if gated else "int8_linear"
    device = _device(x, what)
    if dtype is None:  # that of the first tensor which has one
        dtype = next((t.dtype for t in (None if x.dtype == torch.int8 else x, out, bias, residual) if t is not None),
                     torch.bfloat16)
    code = _DT16.get(dtype)
    if code is None:
        _error(N.UNSUPPORTED_TYPE, f"{what}: {dtype} (float16 and bfloat16 are supported)")
    if stream is not None or device != _current_device():
        rest = (bias,) if gated else (bias, residual)
        return _elsewhere(fn, device, stream, x, w, w_scale, *rest, x_scale=x_scale, activation=activation, dtype=dtype,
                          out=out)
    act = _activation(activation)
    if x.dim() != 2 or w.dim() != 2:
        _error(N.SHAPE_MISMATCH, f"{what}: x and w must be matrices")
    m, k = x.shape
    wide = w.shape[0]
    if gated and wide % 2:
        _error(N.SHAPE_MISMATCH, f"int8_gated_linear: w holds two projections, {wide} rows are not even")
    n = wide // 2 if gated else wide
    if x.dtype == torch.int8:
        if x_scale is None:
            _error(N.INVALID_ARGUMENT, f"{what}: int8 x needs x_scale")
        xsp = _vector(x_scale, m, torch.float32, device, "x_scale")
        ldx = _matrix(x, m, k, torch.int8, device, "x")
        if not xsp:  # no rows
            m = 0
    else:
        if x_scale is not None:
            _error(N.INVALID_ARGUMENT, f"{what}: x_scale belongs to an int8 x")
        xsp = 0
        ldx = _matrix(x, m, k, dtype, device, "x")
    ldw = _matrix(w, wide, k, torch.int8, device, "w")
    wsp = _vector(w_scale, wide, torch.float32, device, "w_scale")
    if out is None:
        out = x.new_empty((m, n), dtype=dtype)
        ldy = n
    else:
        ldy = _matrix(out, m, n, dtype, device, "out")
    bp = 0 if bias is None else _vector(bias, wide, dtype, device, "bias")
    rp = ldr = 0
    if residual is not None:
        ldr = _matrix(residual, m, n, dtype, device, "residual")
        rp = residual.data_ptr()
    xp, wp = x.data_ptr(), w.data_ptr()
    head = (code, act, m, n, k, xp, ldx, xsp, wp, ldw, wsp, bp, rp, ldr, out.data_ptr(), ldy)
    lib = N.lib()
    size = lib.cuopx_int8_gated_linear_workspace_size if gated else lib.cuopx_int8_linear_workspace_size
    wsb = _scratch(size, head)
    ws = x.new_empty(wsb, dtype=torch.uint8) if wsb else None
    call = lib.cuopx_int8_gated_linear if gated else lib.cuopx_int8_linear
    rc = call(_INT8.pack(*head, ws.data_ptr() if wsb else 0, wsb), _raw_stream(device))
    if rc:
        N.check(rc, "cuopx_" + what)
    return out


def int8_linear(x: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, bias: Optional[torch.Tensor] = None,
                residual: Optional[torch.Tensor] = None, *, x_scale: Optional[torch.Tensor] = None,
                activation: str = "none", dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None,
                stream=None) -> torch.Tensor:
    """y = act(x_scale[:, None] * w_scale * (x @ w.T) + bias) + residual (cuopx_int8_linear).

    w: int8 [N, K] and w_scale: float32 [N], as quantize_int8 lays weights out.
    x: [M, K], int8 with x_scale, float32 [M], or float16 or bfloat16, which the
    call quantises row by row.  bias: [N]; residual: [M, N], which may be `out`
    itself; both of `dtype`, float16 or bfloat16, the result's type (x's own, or
    for an int8 x that of out, bias or residual, else bfloat16).  K is at most
    131071.  Integer sums are exact, the rest is fp32, rounded once."""
    return _int8(int8_linear, False, x, w, w_scale, bias, residual, x_scale, activation, dtype, out, stream)


def int8_gated_linear(x: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
                      x_scale: Optional[torch.Tensor] = None, activation: str = "silu",
                      dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None,
                      stream=None) -> torch.Tensor:
    """y = act(g) * u with [g | u] = x_scale[:, None] * w_scale * (x @ w.T) + bias (cuopx_int8_gated_linear).

    w: int8 [2N, K] with the gate's rows first, w_scale: [2N], bias: [2N]; the
    rest as in int8_linear."""
    return _int8(int8_gated_linear, True, x, w, w_scale, bias, None, x_scale, activation, dtype, out, stream)
