"""Orthogonalised updates for torch tensors over the C ABI.

  orthogonalize(g, ...)              the iteration's X for G: singular values towards 1, vectors kept
  muon_step(w, g, momentum, lr=...)  one optimiser step of Muon on a linear layer's weight

Operands are matrices [rows, cols], or stacks of them [batch, rows, cols], whose
rows are contiguous; a stack's matrices may lie side by side in wider rows.
Calls run on their tensors' device and on `stream`, as in layers.py.
"""
from __future__ import annotations

import ctypes as C
import math
from functools import lru_cache
from struct import Struct
from typing import Optional

import torch

from . import _native as N
from .layers import _DT, _current_device, _device, _elsewhere, _error, _raw_stream

# Of the quintic iteration (K. Jordan, "Muon", 2024): five steps take singular
# values from 0.01 on to between 0.7 and 1.2.
COEFFICIENTS = (3.4445, -4.7750, 2.0315)

# The argument structs of include/cuopx.h.
_ORTHO = Struct("=4i3qdQQ2qQ2qQQ")
_MUON = Struct("=6i3qdQ4dQQ2qQ2qQ2qQQ")

_empty = torch.empty


@lru_cache(maxsize=64)
def _coefficients(triples):
    """(a, b, c) of each step as C doubles; triples holds plain floats, so that equal keys are equal numbers."""
    flat = [v for t in triples for v in t]
    return (C.c_double * max(1, len(flat)))(*flat)


def _triple(t):
    a, b, c = t
    return float(a), float(b), float(c)


def _schedule(coefficients, steps: int, what: str):
    if steps < 0:
        _error(N.INVALID_ARGUMENT, f"{what}: {steps} steps")
    triples = None
    try:
        try:
            triples = (_triple(coefficients),) * steps  # one for all steps
        except (TypeError, ValueError, RuntimeError):
            triples = tuple(_triple(t) for t in coefficients)
    except (TypeError, ValueError, RuntimeError):
        pass
    if triples is None or len(triples) != steps:
        _error(N.INVALID_ARGUMENT, f"{what}: coefficients must be (a, b, c), or {steps} of them for {steps} steps")
    return _coefficients(triples)


def _stack(t: torch.Tensor, shape, device: int, what: str):
    """(dtype code, address, leading dimension, stride between matrices) of a stack (checked)."""
    code = _DT.get(t.dtype)
    if code is None or t.get_device() != device:
        _error(N.UNSUPPORTED_TYPE if code is None else N.INVALID_ARGUMENT,
               f"{what} must be float32, float16 or bfloat16 on cuda:{device}, not {t.dtype} on {t.device}")
    if t.shape != shape:
        _error(N.SHAPE_MISMATCH, f"{what} must be {tuple(shape)}, not {tuple(t.shape)}")
    rows, cols = shape[-2:]
    ld, cs = t.stride()[-2:]
    batch = shape[0] if len(shape) == 3 else 1
    stride = t.stride(0) if batch > 1 else 0
    if rows <= 1:
        ld = cols
    if cs != 1 and cols > 1:
        _error(N.INVALID_ARGUMENT, f"{what}: rows must be contiguous (strides {t.stride()})")
    return code, t.data_ptr(), ld, stride


def _bits(operand_bits: Optional[int], result: torch.dtype, what: str) -> int:
    """Bits that the products' operands keep: those asked for, else by the result's type (as in the C call)."""
    if operand_bits is None:
        return 11 if result == torch.bfloat16 else 22
    if operand_bits not in (11, 22):
        _error(N.INVALID_ARGUMENT, f"{what}: operand_bits must be 11, 22 or None, not {operand_bits!r}")
    return int(operand_bits)


def _sizes(t: torch.Tensor, what: str):
    if t.dim() not in (2, 3):
        _error(N.SHAPE_MISMATCH, f"{what} must be a matrix or a stack of matrices")
    shape = t.shape
    return (shape[0] if len(shape) == 3 else 1), shape[-2], shape[-1]


def orthogonalize(g: torch.Tensor, *, steps: int = 5, coefficients=COEFFICIENTS, eps: float = 1e-7,
                  out: Optional[torch.Tensor] = None, operand_bits: Optional[int] = None, stream=None) -> torch.Tensor:
    """X after `steps` times X = a X + (b A + c A A) X, A = X X^T, from g / (||g|| + eps) (cuopx_orthogonalize).

    g: [rows, cols] or [batch, rows, cols], float32, float16 or bfloat16; out:
    the same shape, any of these types (g's by default), or g itself.
    coefficients: (a, b, c), or one such triple for each step; a singular value
    in [0, 1] may not grow beyond 1024 by them.  operand_bits: what the products'
    operands keep, 11 for a bfloat16 result and 22 for others unless given.  With 11
    the result is off by 2e-4 to 2e-3 of its norm, bfloat16's own rounding by 1.7e-3; with 22, which takes up to three times
    as long, by 5e-6 (64 x 3000) to 2e-4 (8192 x 28672): the tensor cores' fp32
    sums, whose error grows with their depth.  X itself keeps 22 bits either way."""
    device = _device(g, "orthogonalize")
    if stream is not None or device != _current_device():
        return _elsewhere(orthogonalize, device, stream, g, steps=steps, coefficients=coefficients, eps=eps, out=out,
                          operand_bits=operand_bits)
    batch, rows, cols = _sizes(g, "g")
    coeff = _schedule(coefficients, steps, "orthogonalize")
    gd, gp, ldg, sg = _stack(g, g.shape, device, "g")
    if out is None:
        out = _empty(g.shape, dtype=g.dtype, device=g.device)
    od, op, ldo, so = _stack(out, g.shape, device, "out")
    lib = N.lib()
    bits = _bits(operand_bits, out.dtype, "orthogonalize")
    wsb = lib.cuopx_orthogonalize_workspace_size_bits(batch, rows, cols, bits)
    ws = _empty(wsb, dtype=torch.uint8, device=g.device) if wsb else None
    rc = lib.cuopx_orthogonalize(
        _ORTHO.pack(gd, od, steps, bits, batch, rows, cols, eps, C.addressof(coeff), gp, ldg, sg, op, ldo, so,
                    ws.data_ptr() if wsb else 0, wsb), _raw_stream(device))
    if rc:
        N.check(rc, "cuopx_orthogonalize")
    return out


def muon_step(w: torch.Tensor, g: torch.Tensor, momentum: torch.Tensor, *, lr: float, mu: float = 0.95,
              weight_decay: float = 0.0, nesterov: bool = True, scale: Optional[float] = None, steps: int = 5,
              coefficients=COEFFICIENTS, eps: float = 1e-7, lr_tensor: Optional[torch.Tensor] = None,
              operand_bits: Optional[int] = None, stream=None) -> torch.Tensor:
    """One step of Muon, in place on w and momentum; returns w (cuopx_muon_step).

      momentum = mu momentum + g;  u = g + mu momentum with nesterov, else momentum
      w = (1 - lr weight_decay) w - lr scale orthogonalize(u)

    w, g, momentum: the same shape, [rows, cols] or [batch, rows, cols], each
    float32, float16 or bfloat16.  scale: 0.2 sqrt(max(rows, cols)) by default,
    which gives the step a root mean square of about 0.2 lr whatever the shape,
    transposed weights too.  lr_tensor, one float32 on the device, multiplies lr when the
    kernel runs, so that a captured graph can follow a schedule.  operand_bits: as in
    orthogonalize, w being the result; 11 makes the steps of float16 and float32 weights as
    fast as bfloat16 weights', each off by 2e-4 to 2e-3 of itself."""
    device = _device(w, "muon_step")
    if stream is not None or device != _current_device():
        return _elsewhere(muon_step, device, stream, w, g, momentum, lr=lr, mu=mu, weight_decay=weight_decay,
                          nesterov=nesterov, scale=scale, steps=steps, coefficients=coefficients, eps=eps,
                          lr_tensor=lr_tensor, operand_bits=operand_bits)
    batch, rows, cols = _sizes(w, "w")
    coeff = _schedule(coefficients, steps, "muon_step")
    wd, wp, ldw, sw = _stack(w, w.shape, device, "w")
    gd, gp, ldg, sg = _stack(g, w.shape, device, "g")
    md, mp, ldm, sm = _stack(momentum, w.shape, device, "momentum")
    lp = 0
    if lr_tensor is not None:
        if lr_tensor.dtype != torch.float32 or lr_tensor.numel() != 1 or lr_tensor.get_device() != device:
            _error(N.INVALID_ARGUMENT, "muon_step: lr_tensor must be one float32 on w's device")
        lp = lr_tensor.data_ptr()
    if scale is None:
        scale = 0.2 * math.sqrt(max(rows, cols, 1))
    lib = N.lib()
    bits = _bits(operand_bits, w.dtype, "muon_step")
    wsb = lib.cuopx_orthogonalize_workspace_size_bits(batch, rows, cols, bits)
    ws = _empty(wsb, dtype=torch.uint8, device=w.device) if wsb else None
    rc = lib.cuopx_muon_step(
        _MUON.pack(wd, gd, md, steps, 1 if nesterov else 0, bits, batch, rows, cols, eps, C.addressof(coeff), lr, mu,
                   weight_decay, scale, lp, wp, ldw, sw, mp, ldm, sm, gp, ldg, sg, ws.data_ptr() if wsb else 0, wsb),
        _raw_stream(device))
    if rc:
        N.check(rc, "cuopx_muon_step")
    return w
