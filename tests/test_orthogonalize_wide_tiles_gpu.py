"""Orthogonalised updates whose symmetric products run on tiles of 512 columns, as those of the largest weights do: wide
and tall, odd numbers of row tiles, one tile to a pair and several, phases of other widths in between."""
import pytest
import torch

import cuop_b200 as cx
import muon22_refs as W
import muon_refs as R
from test_muon_gpu import gen

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32

# By batch and row tiles of 256 these take 512 whether 66 or 74 pairs run at once; the last three have more tiles than pairs.
SHAPES = [(4, 1500, 1610), (4, 1610, 1500), (4, 1700, 1790), (3, 1793, 1661), (3205, 3300), (3300, 3205), (3, 2900, 2901),
          (2, 3700, 3720), (2, 3720, 3700)]


def singular_values(x):
    """By way of the Gram matrix: good to 1e-8 of the largest, which is all that the bounds need, and fast at these sizes."""
    t = x @ x.mT if x.shape[0] <= x.shape[1] else x.mT @ x
    return torch.linalg.eigvalsh(t).clamp_min(0).sqrt()


@pytest.mark.parametrize("bits", [11, 22])
@pytest.mark.parametrize("shape", SHAPES)
def test_wide_tiles(shape, bits, monkeypatch):
    monkeypatch.setattr(torch.linalg, "svdvals", singular_values)
    coefficients = [R.COEFFICIENTS] * (5 if shape[-1] < 2000 else 2)
    g = torch.randn(shape, generator=gen(sum(shape)), device="cuda")
    g = g + 2 * torch.randn(*shape[:-1], 1, generator=gen(1), device="cuda") * torch.randn(shape[-1], generator=gen(2), device="cuda")
    o = cx.orthogonalize(g, steps=len(coefficients), coefficients=coefficients, operand_bits=bits)
    assert cx.last_kernel() == "ortho_out_w512"
    for _ in range(3):
        assert torch.equal(o, cx.orthogonalize(g, steps=len(coefficients), coefficients=coefficients, operand_bits=bits))
    for x, y in zip(g.view(-1, *shape[-2:]), o.view(-1, *shape[-2:])):
        x0 = R.normalised(x)
        off = float(torch.linalg.matrix_norm(y.double() - R.iterate(x0, coefficients)))
        bound = (W.allowed22 if bits == 22 else R.allowed)(x0, coefficients, F32)
        assert off <= bound, (off, bound)


@pytest.mark.parametrize("shape", [(4, 1500, 1610), (3300, 3205)])
def test_step_on_wide_tiles(shape):
    """The optimiser step goes by the same products: its weight is the one that orthogonalize's result gives."""
    w0 = (torch.randn(shape, generator=gen(3), device="cuda") * 0.02).to(BF)
    g = torch.randn(shape, generator=gen(4), device="cuda").to(BF)
    w, m = w0.clone(), torch.zeros(shape, device="cuda")
    cx.muon_step(w, g, m, lr=0.1, mu=0.0, nesterov=False, weight_decay=0.5, scale=2.0)
    assert cx.last_kernel() == "ortho_step_w512" and torch.equal(m, g.float())
    want = 0.95 * w0.double() - 0.2 * cx.orthogonalize(g, out=torch.empty(shape, device="cuda"), operand_bits=11).double()
    # two products and a sum in fp32, and the weight's rounding
    assert ((w.double() - want).abs() <= 2.0 ** -8 * want.abs() + 4 * 2.0 ** -24 * (w0.double().abs() + 1)).all()
