"""int8 layers where a weight has only just been written, and rows beside those that are not numbers."""
import pytest
import torch

import cuop_b200 as cx
import int8_refs as Q
import layer_refs as R
from test_int8_gpu import gen, operands, strided, values

pytestmark = pytest.mark.gpu
BF, HF, I8 = torch.bfloat16, torch.float16, torch.int8

# rows, outputs, depth, and the last kernel: quantised by a launch of its own, whose work the first loads of W overlap;
# by that launch's form for any alignment (an odd depth); copied W; and by the product's kernel itself.
CHAINS = [(24, 520, 1024, "int8_linear_split"), (64, 520, 1024, "int8_linear_split"), (64, 264, 4096, "int8_linear_split"),
          (16, 1000, 2000, "int8_linear_split"), (17, 520, 1001, "int8_linear_split"), (128, 264, 1024, "int8_linear_split"),
          (8, 520, 1024, "int8_linear_split_q"), (300, 520, 2000, "int8_linear_pair_k2"), (700, 1000, 520, "int8_linear_tc2_256x256")]


@pytest.mark.parametrize("aligned_x", [True, False])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("m,n,k,name", CHAINS)
def test_weights_quantised_just_before(m, n, k, name, gated, aligned_x):
    """Weight, activations and product in one chain of dependent launches, over and over on the same buffers: a product
    that read W before the launch that writes it had ended would get the weight of the turn before."""
    g = gen(m + k)
    wide = 2 * n if gated else n
    ldq = (k + 15) // 16 * 16
    q, s = torch.empty(wide, ldq, dtype=I8, device="cuda")[:, :k], torch.empty(wide, device="cuda")
    ws = [torch.randn(k, wide, generator=g, device="cuda").to(BF) * (k ** -0.5 * (i + 1)) for i in range(3)]
    x = values(g, m, k, BF)
    if not aligned_x:
        x = strided(x, 1, 1, 0.0)[0]
    layer = cx.int8_gated_linear if gated else cx.int8_linear
    xq, xs = Q.quantize(x)
    want = []
    for w in ws:
        wq, wsc = Q.quantize(w.t())
        want.append(Q.linear(xq, xs, wq, wsc, None, None, "silu", BF, gated))
    torch.cuda.synchronize()
    out = [torch.empty(m, n, dtype=BF, device="cuda") for _ in range(30)]
    for i in range(30):
        cx.quantize_int8(ws[i % 3], trans=True, out=q, scale=s)
        layer(x, q, s, out=out[i], activation="silu")
    got = cx.last_kernel()
    if gated:
        assert got.startswith("int8_gated_linear_" + ("split_q" if name.endswith("_q") else "split" if m <= 64 else ""))
    else:
        assert got == name
    for i in range(30):
        R.assert_within(out[i], *want[i % 3], f"turn {i}")


@pytest.mark.parametrize("m,n,k", [(1, 512, 256), (8, 264, 1000), (24, 200, 1024), (130, 264, 2048), (300, 520, 512)])
def test_rows_beside_those_that_are_not_numbers(m, n, k):
    """Every row that is finite has its own values, whatever the rows beside it hold."""
    g = gen(11)
    x, wq, ws, b, _ = operands(g, m, n, k, BF, False, True, False)
    x = torch.cat((x, x, x))
    bad = torch.zeros(3 * m, dtype=torch.bool, device="cuda")
    for row, col, v in ((m, 3, float("nan")), (2 * m, k - 1, -float("inf"))):
        x[row, col] = v
        bad[row] = True
    y = cx.int8_linear(x, wq, ws, b)
    assert torch.isnan(y[bad]).all()
    good = x[~bad]
    xq, xs = Q.quantize(good)
    R.assert_within(y[~bad], *Q.linear(xq, xs, wq, ws, b, None, "none", BF, False), "finite rows")


@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("dt", [BF, HF, torch.float32])
@pytest.mark.parametrize("k", [5, 64, 4100])
def test_zeros_of_either_sign(dt, trans, k):
    x = torch.zeros(4, k, device="cuda", dtype=dt)
    x[1] = -0.0
    x[2, 0] = torch.finfo(dt).tiny if dt != HF else 2.0 ** -24
    x[3, k - 1] = 1.0
    q, s = cx.quantize_int8(x.t().contiguous() if trans else x, trans=trans)
    least = torch.tensor(2.0 ** -100, device="cuda").double() / 127
    assert (q[:2] == 0).all() and (s[:2] == least.float()).all()
    top = x[2, 0].double().clamp_min(2.0 ** -100)
    assert float(s[2]) == float((top / 127).float()) and int(q[3, k - 1]) == 127
