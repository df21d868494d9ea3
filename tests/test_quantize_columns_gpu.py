"""Quantisation by columns where CTAs of a cluster have no rows, call after call."""
import pytest
import torch

import cuop_b200 as cx
import int8_refs as Q

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("cols", [70, 4000])
@pytest.mark.parametrize("rows", [1025, 1120, 1281, 1344, 1537, 1568])
def test_ctas_without_rows(rows, cols, dt):
    """Eight shares in whole groups of 32 rows leave the last CTA none: it has nothing to do between reading the others'
    maxima and leaving.  Launches follow one another without a pause, so that shared memory changes hands at once."""
    assert 7 * ((rows + 7) // 8 + 31 & ~31) >= rows
    g = torch.Generator(device="cuda").manual_seed(rows + cols)
    xs = [torch.randn(rows, cols, generator=g, device="cuda").to(dt) for _ in range(3)]
    want = [Q.quantize(x.t()) for x in xs]
    q = [torch.empty(cols, rows, dtype=torch.int8, device="cuda") for _ in range(30)]
    s = [torch.empty(cols, device="cuda") for _ in range(30)]
    for i in range(30):
        cx.quantize_int8(xs[i % 3], trans=True, out=q[i], scale=s[i])
    assert cx.last_kernel() == "quantize_columns"
    for i in range(30):
        assert torch.equal(q[i], want[i % 3][0]) and torch.equal(s[i], want[i % 3][1]), i
