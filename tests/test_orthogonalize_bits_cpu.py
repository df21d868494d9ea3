"""Operand bits of the orthogonalised updates without a GPU: refusals, workspace sizes, and the definitions' bound."""
import ctypes as C

import pytest
import torch

import muon22_refs as W
import muon_refs as R
from cuop_b200 import _native as N
from test_weight_operators_cpu import BAD, ROOM, muon, ortho


@pytest.mark.parametrize("bits", [1, 10, 12, 23, 32, -11])
def test_refusals(bits):
    assert N.lib().cuopx_orthogonalize(ortho(reserved=bits), None) == BAD
    assert N.lib().cuopx_muon_step(muon(reserved=bits), None) == BAD


def test_workspace():
    lib = N.lib()
    for size in ((1, 40, 60), (3, 1000, 200), (1, 300, 5000), (8, 2048, 2048)):
        few, full = (lib.cuopx_orthogonalize_workspace_size_bits(*size, b) for b in (11, 22))
        assert few < full == lib.cuopx_orthogonalize_workspace_size(*size) == lib.cuopx_orthogonalize_workspace_size_bits(*size, 0)
        batch, rows, cols = size
        for kw, need in ((dict(reserved=11), few), (dict(reserved=22), full), (dict(reserved=11, out_dtype=N.F32), few),
                         (dict(out_dtype=N.F32), full), (dict(out_dtype=N.F16), full), (dict(), few)):
            kw.update(batch=batch, rows=rows, cols=cols, ldg=cols, ldo=cols, sg=rows * cols, so=rows * cols)
            assert lib.cuopx_orthogonalize(ortho(wsb=need - 1, **kw), None) == ROOM
        for kw, need in ((dict(reserved=11), few), (dict(reserved=22), full), (dict(reserved=11, wd=N.F32), few), (dict(wd=N.F32), full), (dict(wd=N.F16), full),
                         (dict(), few)):
            kw.update(batch=batch, rows=rows, cols=cols, ldw=cols, ldm=cols, ldg=cols, sw=rows * cols, sm=rows * cols, sg=rows * cols)
            assert lib.cuopx_muon_step(muon(wsb=need - 1, **kw), None) == ROOM
    assert lib.cuopx_orthogonalize_workspace_size_bits(1, 1 << 25, 4, 22) == 0


@pytest.mark.parametrize("shape", [(16, 16), (64, 150), (150, 64), (90, 90)])
def test_bound_of_fp32_sums(shape):
    """An iteration in fp32, 22 bits of its operands kept, is inside the bound, one with operands of 11 bits far outside."""
    g = torch.Generator().manual_seed(sum(shape))
    x0 = R.normalised(torch.randn(shape, generator=g, dtype=torch.float64))
    five = [R.COEFFICIENTS] * 5
    ref = R.iterate(x0, five)

    def cut(v):  # hi + lo
        hi = v.to(torch.float16).float()
        return hi + ((v - hi) * 2048).to(torch.float16).float() / 2048

    x = x0.float()
    x = x.mT if shape[0] > shape[1] else x
    for a, b, c in five:
        x = cut(x)
        t = cut(x @ x.mT)
        x = a * x + cut(b * t + c * (t @ t)) @ x
    x = x.mT if shape[0] > shape[1] else x
    allowed = W.allowed22(x0, five, torch.float32)
    assert float((x.double() - ref).norm()) <= allowed
    assert float((R.rounded_iteration(x0, five) - ref).norm()) > 3 * allowed
