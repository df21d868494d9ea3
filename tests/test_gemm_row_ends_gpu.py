"""C's rows start on 16-byte boundaries and end anywhere: a product writes its M x N elements and nothing else, also
where a row ends inside a 16-byte group."""
import pytest
import torch

import cuop_b200 as cx
from helpers import forced_variant

pytestmark = pytest.mark.gpu

HALF = ("tc2", "tc2_256x512", "tc2_256x128", "tc_128x256", "tc_128x128", "tc_128x128_2cta", "tc_128x64_2cta")
SINGLE = ("tf32x3_128x64", "tf32x3_128x128", "tf32x3_128x128_k2", "tf32x3_256x128_pair", "ffma")


def padded(rows, cols, dtype, batch=1):
    """Rows with at least one 16-byte group of room behind them; NaN everywhere."""
    e = 16 // torch.empty(0, dtype=dtype).element_size()
    ld = (cols + e - 1) // e * e + e
    buf = torch.full((batch * rows * ld + e,), float("nan"), dtype=dtype, device="cuda")
    return buf[:batch * rows * ld].view(batch, rows, ld)[:, :, :cols], buf


@pytest.mark.parametrize("m,n,k", [(300, 3, 128), (130, 61, 72), (257, 133, 200), (64, 262, 64)])
@pytest.mark.parametrize("dtype,variant", [(torch.bfloat16, v) for v in (None,) + HALF] + [(torch.float16, None)]
                         + [(torch.float32, v) for v in (None,) + SINGLE])
def test_gemm_writes_end_where_rows_end(dtype, variant, m, n, k):
    g = torch.Generator(device="cuda").manual_seed(n)
    e = 16 // torch.empty(0, dtype=dtype).element_size()
    if dtype == torch.float32:
        m, k = m + 200, k + 600  # 3xTF32 from 256^3 on
    k = k // e * e
    a = torch.randn(m, k, generator=g, device="cuda").to(dtype)
    b = torch.randn(k, (n + e - 1) // e * e, generator=g, device="cuda").to(dtype)[:, :n]
    ref = a.double() @ b.double()
    for beta in (0.0, 1.0):
        c, buf = padded(m, n, dtype)
        c = c[0]
        if beta:
            c.zero_()
        with forced_variant(variant):
            cx.gemm(a, b, c, beta=beta)
        # sums of k products in fp32 (layer_refs.py), 3xTF32 another 2^-20; one rounding
        size = a.double().abs() @ b.double().abs()
        bound = (k + 8) * 2.0 ** -23 * size + 2.0 ** -20 * size + torch.finfo(dtype).eps / 2 * ref.abs()
        assert ((c.double() - ref).abs() <= bound * 1.01).all(), cx.last_kernel()
        assert int((~torch.isnan(buf)).sum()) == m * n, cx.last_kernel()


@pytest.mark.parametrize("dtype,n", [(torch.bfloat16, 61), (torch.float32, 70), (torch.float32, 301)])
def test_batched_gemm_writes_end_where_rows_end(dtype, n):
    from cuop_b200 import _native as N

    g = torch.Generator(device="cuda").manual_seed(n)
    batch, m, k = 3, 260, 264
    e = 16 // torch.empty(0, dtype=dtype).element_size()
    a = torch.randn(batch, m, k, generator=g, device="cuda").to(dtype)
    b = torch.randn(batch, k, (n + e - 1) // e * e, generator=g, device="cuda").to(dtype)
    c, buf = padded(m, n, dtype, batch)
    code = N.F32 if dtype == torch.float32 else N.BF16
    rc = N.lib().cuopx_gemm_strided_batched(code, 0, 0, m, n, k, 1.0, a.data_ptr(), k, m * k, b.data_ptr(), b.stride(1),
                                            b.stride(0), 0.0, c.data_ptr(), c.stride(1), c.stride(0), batch,
                                            torch.cuda.current_stream().cuda_stream)
    assert rc == N.SUCCESS
    x, y = a.double(), b[:, :, :n].double()
    size = x.abs() @ y.abs()
    bound = (k + 8) * 2.0 ** -23 * size + 2.0 ** -20 * size + torch.finfo(dtype).eps / 2 * (x @ y).abs()
    assert ((c.double() - x @ y).abs() <= bound * 1.01).all(), cx.last_kernel()
    assert int((~torch.isnan(buf)).sum()) == batch * m * n, cx.last_kernel()
