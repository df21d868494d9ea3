"""Orthogonalised updates whose Gram tiles several pairs share, one call after the other on the same workspace: every
warp reads what the other pairs have just stored, and the numbers of the call before lie in the same place."""
import pytest
import torch

import cuop_b200 as cx
import muon_refs as R

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", [(64, 3001), (128, 6136), (3000, 64), (256, 16384), (300, 5000), (20, 70, 1800)])
def test_sums_of_other_pairs(shape):
    g = torch.Generator(device="cuda").manual_seed(sum(shape))
    xs = [torch.randn(shape, generator=g, device="cuda") * 4.0 ** i for i in range(4)]
    xs = [x if i % 2 else x + 3 * torch.randn(*shape[:-1], 1, generator=g, device="cuda") * 4.0 ** i for i, x in enumerate(xs)]
    want = [cx.orthogonalize(x).clone() for x in xs]
    torch.cuda.synchronize()
    for x, w in zip(xs, want):
        for one, got in zip(x.view(-1, *shape[-2:]), w.view(-1, *shape[-2:])):
            x0 = R.normalised(one)
            five = [R.COEFFICIENTS] * 5
            assert float(torch.linalg.matrix_norm(got.double() - R.iterate(x0, five))) <= R.allowed(x0, five, torch.float32)
    out = [torch.empty(shape, device="cuda") for _ in range(40)]
    for i in range(40):
        cx.orthogonalize(xs[i % 4], out=out[i])  # the allocator hands out the same workspace every time
    for i in range(40):
        assert torch.equal(out[i], want[i % 4]), i
