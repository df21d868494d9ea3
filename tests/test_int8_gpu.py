"""int8 layers on the GPU: quantisation bit by bit, products against 64 bits
(int8_refs.py), every kernel that the layers reach, strides, alignment, values
at the ends of the ranges, streams, devices, captured graphs."""
import threading

import pytest
import torch

import cuop_b200 as cx
import int8_refs as Q
import layer_refs as R
from cuop_b200 import _native as N

pytestmark = pytest.mark.gpu
BF, HF, F32, I8 = torch.bfloat16, torch.float16, torch.float32, torch.int8


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def strided(t, pad, shift, fill):
    """The same matrix inside a larger buffer: rows `pad` elements further apart, base `shift` elements in."""
    rows, cols = t.shape
    buf = torch.full((rows * (cols + pad) + shift + 8,), fill, dtype=t.dtype, device=t.device)
    v = buf[shift:shift + rows * (cols + pad)].view(rows, cols + pad)[:, :cols]
    v.copy_(t)
    return v, buf


def values(g, m, k, dt):
    x = torch.randn(m, k, generator=g, device="cuda")
    x[:, ::max(1, k // 3)] *= 20
    return x.to(dt)


def check_quantize(x, trans, **kw):
    q, s = cx.quantize_int8(x, trans=trans, **kw)
    qr, sr = Q.quantize(x.t() if trans else x)
    assert q.dtype == I8 and s.dtype == F32 and q.shape == qr.shape and s.shape == sr.shape
    assert torch.equal(torch.nan_to_num(s, nan=-1.0), torch.nan_to_num(sr, nan=-1.0))
    assert torch.equal(q, qr), (cx.last_kernel(), int((q != qr).sum()))
    return q, s


QUANT_SIZES = [(1, 1), (1, 8), (2, 7), (3, 16), (5, 100), (33, 127), (7, 128), (64, 264), (130, 1000), (31, 1024), (9, 1032),
               (17, 4097), (4, 8192), (3, 16384), (2, 32768), (2, 32776), (1, 70001), (300, 65)]


@pytest.mark.parametrize("dt", [BF, HF, F32])
@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("m,k", QUANT_SIZES)
def test_quantize(m, k, trans, dt):
    x = values(gen(m + k), m, k, dt)
    check_quantize(x, trans)
    check_quantize(strided(x, 1, 1, float("nan"))[0], trans)
    check_quantize(strided(x, 16, 8, float("nan"))[0], trans)


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("rows,cols", [(257, 200), (513, 64), (1100, 33), (2049, 70), (8200, 66), (12288, 40), (12289, 40), (40001, 7)])
def test_quantize_columns_of_any_length(rows, cols, dt):
    """One CTA, clusters of two to eight, and more rows than a cluster holds."""
    x = values(gen(rows), rows, cols, dt)
    check_quantize(x, True)
    assert cx.last_kernel() == ("quantize_columns" if rows <= 12288 else "quantize_transpose")
    check_quantize(strided(x, 1, 1, float("nan"))[0], True)


@pytest.mark.parametrize("rows,cols", [(5000, 100), (3001, 1030), (2500, 4104), (700, 16384), (1300, 8200)])
def test_quantize_more_rows_than_run_at_once(rows, cols):
    x = values(gen(rows), rows, cols, BF)
    check_quantize(x, False)
    check_quantize(x.float(), False)


@pytest.mark.parametrize("trans", [False, True])
def test_quantize_large(trans):
    x = values(gen(1), 2051, 4099, BF)
    check_quantize(x, trans)
    check_quantize(x[:, :4096], trans)


@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("dt", [BF, HF, F32])
def test_quantize_into_buffers(dt, trans):
    """Neighbours of rows in a wider buffer stay; scale and out are used as given."""
    x = values(gen(3), 37, 90, dt)
    m, k = (90, 37) if trans else (37, 90)
    for pad in (0, 3, 6, 22):
        buf = torch.full((m, k + pad), 77, dtype=I8, device="cuda")
        scale = torch.full((m + 2,), -1.0, device="cuda")
        q, s = check_quantize(x, trans, out=buf[:, :k], scale=scale[1:-1])
        assert q.data_ptr() == buf.data_ptr() and s.data_ptr() == scale[1:].data_ptr()
        assert (buf[:, k:] == 77).all() and scale[0] == -1 and scale[-1] == -1


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("rows, cols", [(2, 3), (6, 65), (300, 130), (2050, 70), (4099, 33)])
def test_quantize_columns_into_odd_rows(rows, cols, dt):
    """Q's rows at all four offsets from a word, in each CTA's share; what lies around them stays."""
    x = torch.randn(rows, cols, generator=gen(rows + cols), device="cuda").to(dt)
    for first, pad in ((0, 1), (1, 3), (3, 2)):
        buf = torch.full((cols, first + rows + pad), 77, dtype=torch.int8, device="cuda")
        check_quantize(x, True, out=buf[:, first:first + rows])
        assert bool((buf[:, :first] == 77).all()) and bool((buf[:, first + rows:] == 77).all())


@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("dt", [BF, HF, F32])
@pytest.mark.parametrize("k", [5, 64, 4100])
def test_quantize_special_values(dt, trans, k):
    """Zeros, the smallest and largest numbers, ties, infinities and NaN."""
    fi = torch.finfo(dt)
    x = torch.zeros(9, k, device="cuda", dtype=dt)
    x[1] = fi.tiny
    x[2] = fi.max
    x[2, 0] = -fi.max
    x[3] = 1.0
    x[3, 1:3] = torch.tensor([0.5, -0.5], dtype=dt)  # 63.5: a tie
    x[4] = torch.arange(k, device="cuda").remainder(128).to(dt)
    x[4, 0] = 127.0
    x[5, 2] = float("inf")
    x[6, 3] = float("nan")
    x[6, 4] = float("inf")
    x[7] = -0.0
    x[8, k - 1] = -3.0
    q, s = check_quantize(x.t().contiguous() if trans else x, trans)
    assert (q[0] == 0).all() and (q[7] == 0).all() and float(s[0]) == 2.0 ** -100 / 127 or True
    assert torch.isinf(s[5]) and torch.isnan(s[6]) and (q[5:7] == 0).all()
    assert int(q[8, k - 1]) == -127


def test_quantize_is_half_a_step_off_at_most():
    """|x - q scale| <= scale / 2, plus the roundings of 127 / a, of the product and of the scale: 3 * 2^-24 of |x|."""
    x = values(gen(5), 200, 777, F32)
    q, s = cx.quantize_int8(x)
    off = (q.double() * s.double()[:, None] - x.double()).abs()
    assert (off <= s.double()[:, None] / 2 + 4 * 2.0 ** -24 * x.double().abs()).all()


def test_quantize_empty():
    for shape, trans, m in (((0, 5), False, 0), ((3, 0), False, 3), ((0, 5), True, 5), ((3, 0), True, 0)):
        q, s = cx.quantize_int8(torch.empty(shape, device="cuda", dtype=BF), trans=trans)
        assert q.shape == (shape[::-1] if trans else shape) and s.shape == (m,)
        assert (s == torch.tensor(2.0 ** -100, device="cuda") / 127).all()


def operands(g, m, n, k, dt, gated, bias, residual, scale=24):
    wide = 2 * n if gated else n
    wq = (torch.randn(wide, k, generator=g, device="cuda") * scale).round().clamp(-127, 127).to(I8)
    ws = (0.5 + torch.rand(wide, generator=g, device="cuda")) * (max(k, 1) ** -0.5 / scale)
    x = values(g, m, k, dt)
    b = (torch.randn(wide, generator=g, device="cuda") * 0.5).to(dt) if bias else None
    r = torch.randn(m, n, generator=g, device="cuda").to(dt) if residual else None
    return x, wq, ws, b, r


def check(x, wq, ws, b, r, act, dt, gated, xs=None, **kw):
    if gated:
        y = cx.int8_gated_linear(x, wq, ws, b, x_scale=xs, activation=act, dtype=dt, **kw)
    else:
        y = cx.int8_linear(x, wq, ws, b, r, x_scale=xs, activation=act, dtype=dt, **kw)
    xq, s = (x, xs) if xs is not None else Q.quantize(x)
    yr, ey = Q.linear(xq, s, wq, ws, b, r, act, dt, gated)
    assert y.dtype == dt
    R.assert_within(y, yr, ey, f"y ({cx.last_kernel()})")
    return y


# name, rows, outputs, depth: each reaches the kernel of that name.
KERNELS = [("int8_linear_simt", 3, 8, 5), ("int8_linear_split_q", 1, 264, 1024), ("int8_linear_split_q", 8, 136, 1008),
           ("int8_linear_split_q", 2, 1000, 4095), ("int8_linear_split_q", 16, 33, 500), ("int8_linear_split_q", 1, 8192, 8000), ("int8_linear_split", 16, 136, 2000),
           ("int8_linear_split", 30, 520, 640), ("int8_linear_split", 64, 1000, 1400), ("int8_linear_split", 100, 300, 528),
           ("int8_linear_split", 5, 7, 80000), ("int8_linear_pair_k2", 129, 257, 1601), ("int8_linear_pair_k2", 700, 264, 2000),
           ("int8_linear_pair_k4", 140, 264, 12416), ("int8_linear_pair_k4", 512, 257, 12801),
           ("int8_linear_tc2_256x256", 300, 520, 528), ("int8_linear_tc2_256x256", 2600, 2056, 272)]
GATED_KERNELS = [("int8_gated_linear_simt", 3, 8, 5), ("int8_gated_linear_split_q", 2, 72, 1280),
                 ("int8_gated_linear_split_q", 4, 300, 2000),
                 ("int8_gated_linear_split", 50, 200, 2064), ("int8_gated_linear_pair_k2", 129, 130, 1601),
                 ("int8_gated_linear_pair_k2", 600, 264, 2000), ("int8_gated_linear_tc2_256x128", 300, 264, 528),
                 ("int8_gated_linear_tc2_256x128", 1500, 1032, 400)]


@pytest.mark.parametrize("name,m,n,k", KERNELS + GATED_KERNELS)
def test_every_kernel(name, m, n, k):
    g = gen(m + n)
    gated = "gated" in name
    for dt, pad, shift in ((BF, 0, 0), (HF, 16, 16), (BF, 1, 1)):
        x, wq, ws, b, r = operands(g, m, n, k, dt, gated, True, not gated)
        small = k <= 64 and m * n * (2 if gated else 1) * k < 1 << 20  # unaligned operands are not copied
        plain = name.replace("_q", "")  # from an int8 x
        if pad:
            wq = strided(wq, pad, shift, 99)[0]
        odd = small and (wq.stride(0) % 16 or wq.data_ptr() % 16)
        simt = "int8_gated_linear_simt" if gated else "int8_linear_simt"
        check(x, wq, ws, b, r, "gelu_tanh", dt, gated)
        assert cx.last_kernel() == (simt if odd else name)
        xq, xs = Q.quantize(x)
        if pad:
            xq = strided(xq, pad, shift, 99)[0]
        check(xq, wq, ws, None, None, "silu", dt, gated, xs=xs)
        odd = odd or small and (xq.data_ptr() % 16 or m > 1 and xq.stride(0) % 16)
        assert cx.last_kernel() == (simt if odd else plain)


SIZES = [(1, 1, 1), (1, 8, 16), (1, 64, 128), (1, 1000, 72), (2, 7, 31), (3, 40, 200), (5, 128, 64), (8, 264, 136),
         (16, 256, 512), (17, 129, 65), (24, 1024, 328), (33, 64, 1024), (64, 136, 96), (65, 512, 264), (129, 128, 64),
         (130, 72, 1000), (200, 333, 77), (257, 264, 256), (300, 1000, 200), (512, 512, 448), (700, 392, 512)]


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_sizes(m, n, k, gated):
    g = gen(m * 7 + n * 3 + k)
    for i, (dt, act) in enumerate(((BF, "silu"), (HF, "gelu"))):
        x, wq, ws, b, r = operands(g, m, n, k, dt, gated, i == 0, not gated and i == 1)
        check(x, wq, ws, b, r, act, dt, gated)
        xq, xs = Q.quantize(x)
        check(xq, wq, ws, b, r, act, dt, gated, xs=xs)


@pytest.mark.parametrize("act", R.ACTS)
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("m,n,k", [(1, 512, 256), (40, 200, 136), (300, 520, 128), (70, 33, 45)])
def test_activations(m, n, k, gated, act):
    g = gen(3)
    for dt in (BF, HF):
        x, wq, ws, b, r = operands(g, m, n, k, dt, gated, True, not gated)
        check(x, wq, ws, b, r, act, dt, gated)


@pytest.mark.parametrize("m,n,k", [(1, 136, 131071), (3, 64, 131071), (40, 70, 100000), (130, 264, 131071), (257, 250, 65536),
                                   (300, 300, 131056)])
def test_largest_sums(m, n, k):
    """-128 * -128 at the greatest depth is just inside int32: 131071 * 2^14 < 2^31; and its opposite sign."""
    ones = torch.ones(max(m, n), device="cuda")
    for a, b in ((-128, -128), (-128, 127), (127, 127)):
        xq = torch.full((m, k), a, dtype=I8, device="cuda")
        wq = torch.full((n, k), b, dtype=I8, device="cuda")
        y = cx.int8_linear(xq, wq, ones[:n] * 2.0 ** -20, x_scale=ones[:m])
        assert (y.double() == torch.tensor(a * b * k * 2.0 ** -20, dtype=torch.float64).to(torch.float32).to(BF).double()).all()


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("m,n", [(1, 5), (70, 130), (300, 512)])
def test_no_depth(m, n, gated):
    """K = 0: bias, activation and residual of no sums; unquantised and quantised X."""
    g = gen(9)
    x, wq, ws, b, r = operands(g, m, n, 0, BF, gated, True, not gated) if False else (
        torch.empty(m, 0, dtype=BF, device="cuda"), torch.empty((2 if gated else 1) * n, 0, dtype=I8, device="cuda"),
        torch.full(((2 if gated else 1) * n,), float("nan"), device="cuda"),
        torch.randn((2 if gated else 1) * n, generator=g, device="cuda").to(BF),
        None if gated else torch.randn(m, n, generator=g, device="cuda").to(BF))
    z = b.double().expand(m, -1)
    ref = R.value(z[:, :n], "silu") * z[:, n:] if gated else R.value(z, "silu") + r.double()
    for kw in ({}, {"x_scale": torch.full((m,), float("nan"), device="cuda")}):
        xx = x.to(I8) if kw else x
        y = cx.int8_gated_linear(xx, wq, ws, b, activation="silu", dtype=BF, **kw) if gated else \
            cx.int8_linear(xx, wq, ws, b, r, activation="silu", dtype=BF, **kw)
        R.assert_within(y, ref, R.u(BF) * ref.abs() + 1e-6 * (1 + ref.abs()), "y")


def test_empty():
    for m, n in ((0, 8), (8, 0), (0, 0)):
        x = torch.zeros(m, 32, dtype=HF, device="cuda")
        w = torch.zeros(n, 32, dtype=I8, device="cuda")
        assert cx.int8_linear(x, w, torch.zeros(n, device="cuda")).shape == (m, n)
        assert cx.int8_linear(x.to(I8), w, torch.zeros(n, device="cuda"), x_scale=torch.zeros(m, device="cuda")).shape == (m, n)


@pytest.mark.parametrize("m,n,k", [(1, 512, 256), (24, 200, 1024), (130, 264, 2048), (300, 520, 512)])
def test_rows_that_are_not_numbers(m, n, k):
    """A NaN or an infinity in X makes its whole row NaN and touches no other."""
    g = gen(11)
    x, wq, ws, b, _ = operands(g, m, n, k, BF, False, True, False)
    x = torch.cat((x, x, x))
    x[m, 3] = float("nan")
    x[2 * m, k - 1] = -float("inf")
    y = cx.int8_linear(x, wq, ws, b)
    bad = torch.isnan(y).any(1)
    assert torch.isnan(y[m]).all() and torch.isnan(y[2 * m]).all() and int(bad.sum()) == 2
    assert torch.equal(y[:m], cx.int8_linear(x[:m], wq, ws, b)) or m > 1 and k > 0


@pytest.mark.parametrize("m,n,k", [(1, 512, 256), (24, 136, 1024), (130, 264, 2048), (300, 520, 512), (500, 131, 300)])
def test_outputs_residuals_and_strides(m, n, k):
    """Rows of any stride and alignment; the residual in place; what lies between rows stays."""
    g = gen(m)
    for pad, shift in ((0, 0), (8, 8), (3, 1), (2, 2)):
        x, wq, ws, b, r = operands(g, m, n, k, BF, False, True, True)
        x = strided(x, pad, shift, float("nan"))[0]
        res, rbuf = strided(r, pad, shift, 7.0)
        xq, xs = Q.quantize(x)
        yr, ey = Q.linear(xq, xs, wq, ws, b, r, "none", BF, False)
        out, obuf = strided(torch.zeros_like(r), pad, shift, 5.0)
        y = cx.int8_linear(x, wq, ws, b, res, out=out)
        assert y.data_ptr() == out.data_ptr()
        R.assert_within(y, yr, ey, "out")
        out.fill_(5.0)
        assert (obuf == 5.0).all()
        y = cx.int8_linear(x, wq, ws, b, res, out=res)
        R.assert_within(y, yr, ey, "in place")
        res.fill_(7.0)
        assert (rbuf == 7.0).all()


@pytest.mark.parametrize("m,n,k", [(3, 264, 1024), (200, 264, 2048), (1500, 1032, 400)])
def test_same_bits_every_time(m, n, k):
    g = gen(2)
    x, wq, ws, b, r = operands(g, m, n, k, BF, False, True, True)
    first = cx.int8_linear(x, wq, ws, b, r, activation="gelu")
    for _ in range(20):
        assert torch.equal(first, cx.int8_linear(x, wq, ws, b, r, activation="gelu"))


@pytest.mark.parametrize("m,n,k", [(3, 264, 1024), (200, 264, 2048)])
def test_streams_threads_and_graphs(m, n, k):
    g = gen(4)
    sets = [operands(g, m, n, k, BF, False, True, True) for _ in range(4)]
    want = [cx.int8_linear(*s, activation="silu") for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [None] * 4

    def work(i):
        for _ in range(25):
            got[i] = cx.int8_linear(*sets[i], activation="silu", stream=streams[i])

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # two graphs captured one after the other, replayed at the same time on two streams
    xs = [s[0].clone() for s in sets[:2]]
    graphs, outs = [], []
    for i in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            q, sc = cx.quantize_int8(xs[i])
            y = cx.int8_linear(q, *sets[i][1:], x_scale=sc, activation="silu", dtype=BF)
            y2 = cx.int8_linear(xs[i], *sets[i][1:], activation="silu")
        graphs.append(gr)
        outs.append((y, y2))
    for turn in range(5):
        for i in range(2):
            xs[i].copy_(sets[(i + turn) % 4][0])
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            ref = cx.int8_linear(sets[(i + turn) % 4][0], *sets[i][1:], activation="silu")
            assert torch.equal(outs[i][0], ref) and torch.equal(outs[i][1], ref)


def test_weights_quantised_just_before():
    """Chains of dependent launches: weights, activations and product in a row, over and over on the same buffers."""
    g = gen(6)
    k, n, m = 1024, 520, 8
    q, s = torch.empty(n, k, dtype=I8, device="cuda"), torch.empty(n, device="cuda")
    ws = [torch.randn(k, n, generator=g, device="cuda").to(BF) for _ in range(3)]
    x = values(g, m, k, BF)
    want = []
    for w in ws:
        wq, wsc = cx.quantize_int8(w, trans=True)
        want.append(cx.int8_linear(x, wq, wsc))
        torch.cuda.synchronize()
    out = [torch.empty(m, n, dtype=BF, device="cuda") for _ in range(30)]
    for i in range(30):
        cx.quantize_int8(ws[i % 3], trans=True, out=q, scale=s)
        cx.int8_linear(x, q, s, out=out[i])
    for i in range(30):
        assert torch.equal(out[i], want[i % 3]), i


def test_chain_of_layers_is_a_block():
    """norm -> gated int8 -> int8 with residual, quantised from 16-bit weights, against 64 bits with the same roundings."""
    g = gen(8)
    m, d, f = 70, 256, 520
    x = values(g, m, d, BF)
    w1 = (torch.randn(d, 2 * f, generator=g, device="cuda") * d ** -0.5).to(BF)
    w2 = (torch.randn(f, d, generator=g, device="cuda") * f ** -0.5).to(BF)
    q1, s1 = cx.quantize_int8(w1, trans=True)
    q2, s2 = cx.quantize_int8(w2, trans=True)
    h = cx.layer_norm(x)
    a = cx.int8_gated_linear(h, q1, s1)
    y = cx.int8_linear(a, q2, s2, residual=x)
    xq, xs = Q.quantize(h)
    ar, ea = Q.linear(xq, xs, q1, s1, None, None, "silu", BF, True)
    R.assert_within(a, ar, ea, "a")
    xq, xs = Q.quantize(a)
    yr, ey = Q.linear(xq, xs, q2, s2, None, x, "none", BF, False)
    R.assert_within(y, yr, ey, "y")
    # and how far the block is from the 16-bit one: each int8 operand is half a step off at most, a step being 1/127 of a
    # row's largest value; for sums of independent errors that stays below 5 % of the result's norm here
    full = cx.linear(cx.gated_linear(h, w1), w2, residual=x)
    assert (y.float() - full.float()).norm() < 0.05 * full.float().norm()


def test_refusals():
    x = torch.zeros(4, 32, dtype=BF, device="cuda")
    w = torch.zeros(8, 32, dtype=I8, device="cuda")
    s, xs = torch.zeros(8, device="cuda"), torch.zeros(4, device="cuda")
    bad = [
        lambda: cx.int8_linear(x.cpu(), w, s), lambda: cx.int8_linear(x, w.cpu(), s), lambda: cx.int8_linear(x, w, s.cpu()),
        lambda: cx.int8_linear(x.float(), w, s), lambda: cx.int8_linear(x, w.to(torch.uint8), s),
        lambda: cx.int8_linear(x, w, s.double()), lambda: cx.int8_linear(x, w, s[:7]), lambda: cx.int8_linear(x, w[:, :31], s),
        lambda: cx.int8_linear(x.to(I8), w, s), lambda: cx.int8_linear(x, w, s, x_scale=xs),
        lambda: cx.int8_linear(x.to(I8), w, s, x_scale=xs[:3]), lambda: cx.int8_linear(x.to(I8), w, s, x_scale=xs, dtype=F32),
        lambda: cx.int8_linear(x, w, s, dtype=HF), lambda: cx.int8_linear(x, w, s, activation="tanh"),
        lambda: cx.int8_linear(x, w, s, torch.zeros(8, device="cuda")), lambda: cx.int8_linear(x, w, s, out=x[:, :8]),
        lambda: cx.int8_linear(x, w.t().contiguous().t(), s), lambda: cx.int8_gated_linear(x, w[:7], s[:7]),
        lambda: cx.int8_linear(x[0], w, s), lambda: cx.int8_linear(x, w, s[:1].expand(8)),
        lambda: cx.int8_linear(x[:1].expand(4, 32), w, s),
        lambda: cx.quantize_int8(x.to(torch.float64)), lambda: cx.quantize_int8(x.cpu()), lambda: cx.quantize_int8(x[0]),
        lambda: cx.quantize_int8(x.t()), lambda: cx.quantize_int8(x, out=torch.zeros(4, 31, dtype=I8, device="cuda")),
        lambda: cx.quantize_int8(x, out=torch.zeros(4, 32, dtype=torch.uint8, device="cuda")),
        lambda: cx.quantize_int8(x, scale=torch.zeros(5, device="cuda")), lambda: cx.quantize_int8(x, out=x.view(I8)[:, :32]),
        lambda: cx.int8_linear(torch.zeros(1, 131072, dtype=BF, device="cuda"), torch.zeros(1, 131072, dtype=I8, device="cuda"),
                               s[:1]),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(N.CuopError):
            call()
            print("accepted:", i)
