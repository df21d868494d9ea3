"""Feed-forward layer operators for torch tensors over the C ABI.

  linear(x, w, ...)          y = act(x w + bias) + residual
  gated_linear(x, w, ...)    y = act(x w_gate + b_gate) * (x w_up + b_up)
  layer_norm(x, ...)         y = (x - mean) / sqrt(var + eps) * weight + bias
  dropout(x, p, seed, ...)   y = (keep ? x / (1 - p) : 0) + residual

and their gradients as calls of their own (linear_backward, ...): like the
other operators these work on raw device memory and record nothing for
autograd.  Matrices are row-major 2-D tensors with unit column stride and any
row stride of at least their width.

Every call runs on its tensors' device, on `stream` or else on that device's
current stream; results and scratch are allocated on the same stream.
"""
from __future__ import annotations

from struct import Struct
from typing import Optional

import torch

from . import _native as N

_DT16 = {torch.float16: N.F16, torch.bfloat16: N.BF16}
_DT = {torch.float32: N.F32, torch.float16: N.F16, torch.bfloat16: N.BF16}
_ACT = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4, "sigmoid": 5}

# The argument structs of include/cuopx.h.
_LINEAR = Struct("=4i3qQqQqQQqQqQqQQ")
_LINEAR_BACKWARD = Struct("=4i3qQqQqQqQqQqQqQQQ")
_NORM = Struct("=2i2qdQqQQQqQQQqQqQQQQ")
_DROPOUT = Struct("=2i2qdQQQQqQqQq")

_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice
_empty = torch.empty


def _error(code: int, what: str):
    raise N.CuopError(code, what)


def _elsewhere(fn, device: int, stream, *args, **kwargs):
    """fn(*args, **kwargs) with `device` and `stream` (None: the device's current one) made current."""
    with torch.cuda.device(device):
        if stream is None:
            return fn(*args, **kwargs)
        if not isinstance(stream, torch.cuda.Stream):
            handle = int(stream)
            stream = torch.cuda.ExternalStream(handle, device=device) if handle else torch.cuda.default_stream(device)
        if stream.device.index != device:
            _error(N.INVALID_ARGUMENT, f"stream of {stream.device} for tensors on cuda:{device}")
        with torch.cuda.stream(stream):
            return fn(*args, **kwargs)


def _device(t: torch.Tensor, what: str) -> int:
    d = t.get_device()
    if d < 0:
        _error(N.INVALID_ARGUMENT, f"{what}: tensor is not on a CUDA device (no CPU path exists)")
    return d


def _matrix(t: torch.Tensor, rows: int, cols: int, dtype, device: int, what: str) -> int:
    """Leading dimension of a rows x cols operand (checked)."""
    if t.dtype != dtype or t.get_device() != device:
        _error(N.UNSUPPORTED_TYPE if t.dtype != dtype else N.INVALID_ARGUMENT,
               f"{what} must be {dtype} on cuda:{device}, not {t.dtype} on {t.device}")
    shape = t.shape
    if len(shape) != 2 or shape[0] != rows or shape[1] != cols:
        _error(N.SHAPE_MISMATCH, f"{what} must be {rows} x {cols}, not {tuple(shape)}")
    ld, cs = t.stride()
    if rows <= 1:
        ld = cols
    if (cs != 1 and cols > 1) or ld < cols:
        _error(N.INVALID_ARGUMENT, f"{what}: rows must be contiguous and must not overlap (strides {t.stride()})")
    return ld


def _vector(t: torch.Tensor, n: int, dtype, device: int, what: str) -> int:
    """Address of a contiguous vector of n elements (checked)."""
    if t.dtype != dtype or t.get_device() != device:
        _error(N.UNSUPPORTED_TYPE if t.dtype != dtype else N.INVALID_ARGUMENT,
               f"{what} must be {dtype} on cuda:{device}, not {t.dtype} on {t.device}")
    if t.dim() != 1 or t.shape[0] != n or (n > 1 and t.stride(0) != 1):
        _error(N.SHAPE_MISMATCH, f"{what} must be a contiguous vector of {n}, not {tuple(t.shape)}")
    return t.data_ptr()


def _activation(name: str) -> int:
    code = _ACT.get(name)
    if code is None:
        _error(N.INVALID_ARGUMENT, f"unknown activation {name!r} (known: {', '.join(_ACT)})")
    return code


def _linear(fn, gated: bool, x, w, bias, residual, activation, trans_w, out, preact, stream):
    what = "gated_linear" if gated else "linear"
    dtype = x.dtype
    code = _DT16.get(dtype)
    device = _device(x, what)
    if code is None:
        _error(N.UNSUPPORTED_TYPE, f"{what}: {dtype} (float16 and bfloat16 are supported)")
    if stream is not None or device != _current_device():
        rest = (bias,) if gated else (bias, residual)
        return _elsewhere(fn, device, stream, x, w, *rest, activation=activation, trans_w=trans_w, out=out,
                          preact=preact)
    act = _activation(activation)
    if x.dim() != 2 or w.dim() != 2:
        _error(N.SHAPE_MISMATCH, f"{what}: x and w must be matrices")
    m, k = x.shape
    wide = w.shape[0] if trans_w else w.shape[1]
    if gated and wide % 2:
        _error(N.SHAPE_MISMATCH, f"gated_linear: w holds two projections, {wide} columns are not even")
    n = wide // 2 if gated else wide
    ldx = _matrix(x, m, k, dtype, device, "x")
    ldw = _matrix(w, wide, k, dtype, device, "w") if trans_w else _matrix(w, k, wide, dtype, device, "w")
    if out is None:
        out = x.new_empty((m, n))
        ldy = n
    else:
        ldy = _matrix(out, m, n, dtype, device, "out")
    bp = 0 if bias is None else _vector(bias, wide, dtype, device, "bias")
    rp = ldr = zp = ldz = 0
    if residual is not None:
        ldr = _matrix(residual, m, n, dtype, device, "residual")
        rp = residual.data_ptr()
    if preact is not None:
        ldz = _matrix(preact, m, wide, dtype, device, "preact")
        zp = preact.data_ptr()
    xp, wp, yp = x.data_ptr(), w.data_ptr(), out.data_ptr()
    head = (code, 1 if trans_w else 0, act, 0, m, n, k, xp, ldx, wp, ldw, bp, rp, ldr, yp, ldy, zp, ldz)
    lib = N.lib()
    ws = None
    wsp = wsb = 0
    if (xp | wp | yp | zp) & 15 or (ldx | ldw | ldy | ldz | n) & 7:  # the calls that may want a workspace
        size = lib.cuopx_gated_linear_workspace_size if gated else lib.cuopx_linear_workspace_size
        wsb = size(_LINEAR.pack(*head, 0, 0))
        if wsb:
            ws = _empty(wsb, dtype=torch.uint8, device=x.device)
            wsp = ws.data_ptr()
    call = lib.cuopx_gated_linear if gated else lib.cuopx_linear
    rc = call(_LINEAR.pack(*head, wsp, wsb), _raw_stream(device))
    if rc:
        N.check(rc, "cuopx_gated_linear" if gated else "cuopx_linear")
    return out


def linear(x: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor] = None,
           residual: Optional[torch.Tensor] = None, *, activation: str = "none", trans_w: bool = False,
           out: Optional[torch.Tensor] = None, preact: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """y = act(x op(w) + bias) + residual, in one kernel (cuopx_linear).

    x: [M, K]; w: [K, N], or [N, K] with trans_w; bias: [N]; residual: [M, N],
    which may be `out` itself; float16 or bfloat16.  preact, a [M, N] tensor,
    receives x op(w) + bias for linear_backward.  activation: "none", "relu",
    "gelu", "gelu_tanh", "silu" or "sigmoid"."""
    return _linear(linear, False, x, w, bias, residual, activation, trans_w, out, preact, stream)


def gated_linear(x: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor] = None, *, activation: str = "silu",
                 trans_w: bool = False, out: Optional[torch.Tensor] = None, preact: Optional[torch.Tensor] = None,
                 stream=None) -> torch.Tensor:
    """y = act(g) * u with [g | u] = x op(w) + bias, in one kernel (cuopx_gated_linear).

    w: [K, 2N] with the gate's columns first, or [2N, K] with trans_w; bias:
    [2N]; preact, a [M, 2N] tensor, receives [g | u] for gated_linear_backward."""
    return _linear(gated_linear, True, x, w, bias, None, activation, trans_w, out, preact, stream)


def _linear_backward(fn, gated: bool, dy, x, w, preact, activation, trans_w, need_dx, need_dw, need_db, stream):
    what = "gated_linear_backward" if gated else "linear_backward"
    dtype = dy.dtype
    code = _DT16.get(dtype)
    device = _device(dy, what)
    if code is None:
        _error(N.UNSUPPORTED_TYPE, f"{what}: {dtype} (float16 and bfloat16 are supported)")
    if stream is not None or device != _current_device():
        return _elsewhere(fn, device, stream, dy, x, w, preact, activation=activation, trans_w=trans_w,
                          need_dx=need_dx, need_dw=need_dw, need_db=need_db)
    act = _activation(activation)
    if dy.dim() != 2 or x.dim() != 2:
        _error(N.SHAPE_MISMATCH, f"{what}: dy and x must be matrices")
    m, n = dy.shape
    k = x.shape[1]
    wide = 2 * n if gated else n
    lddy = _matrix(dy, m, n, dtype, device, "dy")
    ldx = _matrix(x, m, k, dtype, device, "x")
    w_shape = (wide, k) if trans_w else (k, wide)
    ldw = _matrix(w, *w_shape, dtype, device, "w")
    zp = ldz = 0
    if preact is not None:
        ldz = _matrix(preact, m, wide, dtype, device, "preact")
        zp = preact.data_ptr()
    elif gated or act:
        _error(N.INVALID_ARGUMENT, f"{what}: the forward pass's preact is needed")
    dev = dy.device
    dx = dy.new_empty((m, k)) if need_dx else None
    dw = dy.new_empty(w_shape) if need_dw else None
    db = dy.new_empty(wide) if need_db else None
    head = (code, 1 if trans_w else 0, act, 0, m, n, k, dy.data_ptr(), lddy, x.data_ptr(), ldx, w.data_ptr(), ldw, zp,
            ldz, dx.data_ptr() if need_dx else 0, k, dw.data_ptr() if need_dw else 0, w_shape[1],
            db.data_ptr() if need_db else 0)
    lib = N.lib()
    size = lib.cuopx_gated_linear_backward_workspace_size if gated else lib.cuopx_linear_backward_workspace_size
    wsb = size(_LINEAR_BACKWARD.pack(*head, 0, 0))
    ws = _empty(wsb, dtype=torch.uint8, device=dev) if wsb else None
    call = lib.cuopx_gated_linear_backward if gated else lib.cuopx_linear_backward
    rc = call(_LINEAR_BACKWARD.pack(*head, ws.data_ptr() if wsb else 0, wsb), _raw_stream(device))
    if rc:
        N.check(rc, "cuopx_" + what)
    return dx, dw, db


def linear_backward(dy: torch.Tensor, x: torch.Tensor, w: torch.Tensor, preact: Optional[torch.Tensor] = None, *,
                    activation: str = "none", trans_w: bool = False, need_dx: bool = True, need_dw: bool = True,
                    need_db: bool = True, stream=None):
    """(dx, dw, db) of linear(x, w, bias, residual, ...) for dy, the gradient
    of its result; None where not needed.  preact is what linear stored (not
    needed for activation "none").  The residual's gradient is dy."""
    return _linear_backward(linear_backward, False, dy, x, w, preact, activation, trans_w, need_dx, need_dw, need_db,
                            stream)


def gated_linear_backward(dy: torch.Tensor, x: torch.Tensor, w: torch.Tensor, preact: torch.Tensor, *,
                          activation: str = "silu", trans_w: bool = False, need_dx: bool = True, need_dw: bool = True,
                          need_db: bool = True, stream=None):
    """(dx, dw, db) of gated_linear(x, w, bias, ...) for dy, the gradient of its
    result; dw and db are packed like w and bias."""
    return _linear_backward(gated_linear_backward, True, dy, x, w, preact, activation, trans_w, need_dx, need_dw,
                            need_db, stream)


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, *,
               eps: float = 1e-5, out: Optional[torch.Tensor] = None, mean: Optional[torch.Tensor] = None,
               rstd: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """Layer norm of each row of x [rows, cols] (cuopx_layer_norm); float32,
    float16 or bfloat16.  weight and bias: [cols], of x's type or float32.
    mean and rstd, float32 vectors of `rows`, receive the statistics for
    layer_norm_backward.  out may be x itself."""
    dtype = x.dtype
    code = _DT.get(dtype)
    device = _device(x, "layer_norm")
    if code is None:
        _error(N.UNSUPPORTED_TYPE, f"layer_norm: {dtype}")
    if stream is not None or device != _current_device():
        return _elsewhere(layer_norm, device, stream, x, weight, bias, eps=eps, out=out, mean=mean, rstd=rstd)
    if x.dim() != 2:
        _error(N.SHAPE_MISMATCH, "layer_norm: x must be a matrix")
    rows, cols = x.shape
    ldx = _matrix(x, rows, cols, dtype, device, "x")
    wdtype = weight.dtype if weight is not None else bias.dtype if bias is not None else dtype
    if wdtype != dtype and wdtype != torch.float32:
        _error(N.UNSUPPORTED_TYPE, f"layer_norm: weight of {wdtype} for x of {dtype}")
    wp = 0 if weight is None else _vector(weight, cols, wdtype, device, "weight")
    bp = 0 if bias is None else _vector(bias, cols, wdtype, device, "bias")
    if out is None:
        out = x.new_empty((rows, cols))
        ldy = cols
    else:
        ldy = _matrix(out, rows, cols, dtype, device, "out")
    mp = 0 if mean is None else _vector(mean, rows, torch.float32, device, "mean")
    rp = 0 if rstd is None else _vector(rstd, rows, torch.float32, device, "rstd")
    rc = N.lib().cuopx_layer_norm(
        _NORM.pack(code, _DT[wdtype], rows, cols, eps, x.data_ptr(), ldx, wp, bp, out.data_ptr(), ldy, mp, rp, 0, 0, 0,
                   0, 0, 0, 0, 0), _raw_stream(device))
    if rc:
        N.check(rc, "cuopx_layer_norm")
    return out


def layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor,
                        weight: Optional[torch.Tensor] = None, *, need_dx: bool = True, need_dw: bool = True,
                        need_db: bool = True, stream=None):
    """(dx, dweight, dbias) of layer_norm(x, weight, bias) for dy; None where
    not needed.  mean and rstd are what layer_norm stored; without a weight it
    counts as ones and the two sums are of x's type."""
    dtype = x.dtype
    code = _DT.get(dtype)
    device = _device(x, "layer_norm_backward")
    if code is None:
        _error(N.UNSUPPORTED_TYPE, f"layer_norm_backward: {dtype}")
    if stream is not None or device != _current_device():
        return _elsewhere(layer_norm_backward, device, stream, dy, x, mean, rstd, weight, need_dx=need_dx,
                          need_dw=need_dw, need_db=need_db)
    if x.dim() != 2:
        _error(N.SHAPE_MISMATCH, "layer_norm_backward: x must be a matrix")
    rows, cols = x.shape
    ldx = _matrix(x, rows, cols, dtype, device, "x")
    lddy = _matrix(dy, rows, cols, dtype, device, "dy")
    wdtype = weight.dtype if weight is not None else dtype
    if wdtype != dtype and wdtype != torch.float32:
        _error(N.UNSUPPORTED_TYPE, f"layer_norm_backward: weight of {wdtype} for x of {dtype}")
    wp = 0 if weight is None else _vector(weight, cols, wdtype, device, "weight")
    mp = _vector(mean, rows, torch.float32, device, "mean")
    rp = _vector(rstd, rows, torch.float32, device, "rstd")
    dev = x.device
    dx = x.new_empty((rows, cols)) if need_dx else None
    dw = _empty(cols, dtype=wdtype, device=dev) if need_dw else None
    db = _empty(cols, dtype=wdtype, device=dev) if need_db else None
    head = (code, _DT[wdtype], rows, cols, 0.0, x.data_ptr(), ldx, wp, 0, 0, 0, mp, rp, dy.data_ptr(), lddy,
            dx.data_ptr() if need_dx else 0, cols, dw.data_ptr() if need_dw else 0, db.data_ptr() if need_db else 0)
    lib = N.lib()
    wsb = lib.cuopx_layer_norm_backward_workspace_size(_NORM.pack(*head, 0, 0))
    ws = _empty(wsb, dtype=torch.uint8, device=dev) if wsb else None
    rc = lib.cuopx_layer_norm_backward(_NORM.pack(*head, ws.data_ptr() if wsb else 0, wsb), _raw_stream(device))
    if rc:
        N.check(rc, "cuopx_layer_norm_backward")
    return dx, dw, db


def _rows(t: torch.Tensor, what: str):
    """(rows, cols, ld) of a contiguous tensor of any shape, as one row, or of a row-strided matrix."""
    if t.is_contiguous():
        n = t.numel()
        return 1, n, n
    if t.dim() != 2 or (t.stride(1) != 1 and t.shape[1] > 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
        _error(N.INVALID_ARGUMENT, f"dropout: {what} must be contiguous, or a matrix with contiguous rows")
    return t.shape[0], t.shape[1], t.stride(0) if t.shape[0] > 1 else t.shape[1]


def dropout(x: torch.Tensor, p: float, seed: int, offset: int = 0, *, residual: Optional[torch.Tensor] = None,
            out: Optional[torch.Tensor] = None, offset_tensor: Optional[torch.Tensor] = None,
            stream=None) -> torch.Tensor:
    """y = (keep ? x / (1 - p) : 0) + residual (cuopx_dropout); float32, float16
    or bfloat16.  The mask depends on (seed, offset) and each element's index
    in x alone, and is never stored; a call uses ceil(x.numel() / 4) values of
    `offset`.  offset_tensor, an int64 tensor of one element on the device, is
    added to offset when the kernel runs, so that a captured graph can draw a
    new mask at each replay.  out may be x or residual itself."""
    dtype = x.dtype
    code = _DT.get(dtype)
    device = _device(x, "dropout")
    if code is None:
        _error(N.UNSUPPORTED_TYPE, f"dropout: {dtype}")
    if stream is not None or device != _current_device():
        return _elsewhere(dropout, device, stream, x, p, seed, offset, residual=residual, out=out,
                          offset_tensor=offset_tensor)
    if out is None:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
    rp = op = 0
    rows, cols, ldx = _rows(x, "x")
    same = [out] if residual is None else [out, residual]
    for t in same:
        if t.dtype != dtype or t.get_device() != device or t.shape != x.shape:
            _error(N.SHAPE_MISMATCH, "dropout: out and residual must have x's shape, type and device")
    lds = [_rows(t, "out or residual") for t in same]
    if any(r != rows for r, _, _ in lds):  # one strided operand: all of them as matrices
        rows, cols = x.shape
        ldx = x.stride(0)
        lds = [(rows, cols, t.stride(0)) for t in same]
    if residual is not None:
        rp = residual.data_ptr()
    if offset_tensor is not None:
        if offset_tensor.dtype != torch.int64 or offset_tensor.numel() != 1 or offset_tensor.get_device() != device:
            _error(N.INVALID_ARGUMENT, "dropout: offset_tensor must be one int64 on x's device")
        op = offset_tensor.data_ptr()
    rc = N.lib().cuopx_dropout(
        _DROPOUT.pack(code, 0, rows, cols, p, seed & 0xFFFFFFFFFFFFFFFF, offset & 0xFFFFFFFFFFFFFFFF, op, x.data_ptr(),
                      ldx, rp, lds[1][2] if rp else 0, out.data_ptr(), lds[0][2]), _raw_stream(device))
    if rc:
        N.check(rc, "cuopx_dropout")
    return out


def dropout_backward(dy: torch.Tensor, p: float, seed: int, offset: int = 0, *, out: Optional[torch.Tensor] = None,
                     offset_tensor: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """Gradient of dropout(x, p, seed, offset, ...) with respect to x: the same
    mask and factor on dy.  The residual's gradient is dy."""
    return dropout(dy, p, seed, offset, out=out, offset_tensor=offset_tensor, stream=stream)
