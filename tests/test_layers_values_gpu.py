"""Layer operators at values and in layouts where formulas and checks can go wrong: infinite and vanishing
pre-activations, the activations' tails, results beside their inputs in one buffer, single rows through the tensor
cores, in-place gradients.  Tolerances are those of layer_refs.py unless a test derives its own."""
import math

import pytest
import torch

import cuop_b200 as cx
import layer_refs as R
from cuop_b200 import _native as N
from cuop_b200 import layers as L

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
INF = float("inf")


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rnd(g, *shape, scale=1.0, dtype=BF):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


# ------------------------------------------------------------------ infinite and very large kept pre-activations
@pytest.mark.parametrize("act", R.ACTS)
@pytest.mark.parametrize("dt,big", [(HF, 65504.0), (BF, 1e30)])
@pytest.mark.parametrize("vec", [True, False])
def test_backward_of_infinite_and_very_large_pre_activations(act, dt, big, vec):
    """One row, so that db is dZ.  A kept infinity counts as 3e38: act and act' have their limits there, and a factor
    that has vanished (dY, act', act) makes 0 of it."""
    zs = [-INF, -big, -300.0, -20.0, 0.0, 1.5, 20.0, 300.0, big, INF]
    us = [-INF, -big, -1.5, 0.0, 2.0, big, INF]
    gs = [0.0, 0.5, -0.25, 1024.0]
    rows = [(g, z, u) for g in gs for z in zs for u in us]
    while len(rows) % 8 != (0 if vec else 3):
        rows.append((1.0, 1.0, 1.0))
    n = len(rows)
    dy, z, up = (torch.tensor([[r[i] for r in rows]], device="cuda").to(dt) for i in range(3))
    g, a, b = (t.double().clamp(-3e38, 3e38)[0] for t in (dy, z, up))
    value, slope = R.value(a, act), R.slope(a, act)
    x, kept = torch.ones(1, 8, dtype=dt, device="cuda"), torch.cat((z, up), 1)
    db = cx.gated_linear_backward(dy, x, torch.ones(8, 2 * n, dtype=dt, device="cuda"), kept, activation=act,
                                  need_dx=False, need_dw=False)[2]
    one = cx.linear_backward(dy, x, torch.ones(8, n, dtype=dt, device="cuda"), z, activation=act, need_dx=False, need_dw=False)[2]
    # act_error grows with z without limit, act and act' are at their limits beyond 300
    near = a.clamp(-300, 300)
    rel, floor = 3 * R.act_error(near, act) + 2.0 ** -21, R.act_floor(near, act)
    for what, got, ref, factor in (("dg", db[:n], g * (b * slope), (g * b).abs()), ("du", db[n:], g * value, g.abs()),
                                   ("linear", one, g * slope, g.abs())):
        assert not torch.isnan(got).any(), (what, [rows[i] for i in torch.isnan(got).nonzero()[:3, 0].tolist()])
        ok = (got == ref.to(dt)) | ((got.double() - ref).abs() <= (R.u(dt) + rel) * ref.abs() + floor * factor + 4 * R.TINY[dt])
        assert ok.all(), (what, [(rows[i], got[i].item(), ref[i].item()) for i in (~ok).nonzero()[:5, 0].tolist()])


@pytest.mark.parametrize("act", ["relu", "gelu", "gelu_tanh", "silu", "sigmoid"])
@pytest.mark.parametrize("m,n,k", [(3, 40, 24), (70, 136, 264), (300, 264, 136)])
def test_gated_backward_stays_finite_where_the_forward_pass_does(act, m, n, k):
    """fp16 gates below -65504 are kept as -inf; the forward result there is finite, and so are all three gradients."""
    g = gen(7)
    x, dy = rnd(g, m, k, dtype=HF), rnd(g, m, n, dtype=HF)
    w = rnd(g, k, 2 * n, scale=k ** -0.5, dtype=HF)
    z = rnd(g, m, 2 * n, dtype=HF)
    z[1, :n] = -INF
    z[m - 1, 3] = -INF
    got = cx.gated_linear_backward(dy, x, w, z, activation=act)
    # the definition at -65504: every activation and derivative is 0 there, to 64 bits
    ref = R.linear_backward(dy, x, w, z.clamp_min(-65504.0), act, False, True)
    # act_error grows without limit there while act stays 0: the bounds are those of z = 0 in the same places, whose
    # terms are larger than the zeros', and the last rounding of this sum
    calm = R.linear_backward(dy, x, w, torch.where(z < -1e4, torch.zeros_like(z), z), act, False, True)
    for name, t, (r, _), (_, bound) in zip(("dx", "dw", "db"), got, ref, calm):
        assert torch.isfinite(t).all(), name
        R.assert_within(t, r, bound + R.u(HF) * r.abs(), name)


# ------------------------------------------------------------------ sigmoids in the tails
def spread(lo, hi, dt, count=4096):
    return torch.linspace(lo, hi, count, device="cuda", dtype=torch.float64).to(dt).unique()


@pytest.mark.parametrize("act,dt,far", [("sigmoid", BF, 86.0), ("sigmoid", HF, 17.0), ("silu", BF, 86.0), ("silu", HF, 17.0),
                                        ("gelu_tanh", BF, 9.9), ("gelu_tanh", HF, 5.0)])
def test_sigmoid_slopes_keep_their_relative_accuracy(act, dt, far):
    """s' = s (1 - s) and the slopes made of it, to act_error relative (of their terms), as far as the exponential stays
    a normal fp32 number (its argument below 87)."""
    z = spread(-far, far, dt)[None]
    n = z.shape[1]
    one = torch.ones(1, n, dtype=dt, device="cuda")
    got = cx.linear_backward(one, one[:, :8], torch.ones(8, n, dtype=dt, device="cuda"), z, activation=act, need_dx=False,
                             need_dw=False)[2]
    zz = z.double()[0]
    if act == "gelu_tanh":
        c = 2 * math.sqrt(2 / math.pi)
        arg, inner = c * (zz + 0.044715 * zz ** 3), c * (1 + 0.134145 * zz ** 2)
    else:
        arg, inner = zz, torch.ones_like(zz)
    s, d = torch.sigmoid(arg), torch.sigmoid(arg) * torch.sigmoid(-arg) * inner
    ref, size = (d, d) if act == "sigmoid" else (s + zz * d, s + (zz * d).abs())
    R.assert_within(got, ref, R.u(dt) * ref.abs() + 1.01 * (2 * R.act_error(zz, act) + 2.0 ** -22) * size + R.TINY[dt])


# ------------------------------------------------------------------ gelu in the tails
@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("rows", [16, 1024])
def test_gelu_keeps_its_relative_accuracy_in_the_tails(dt, rows):
    """z Phi(z) and its derivative to act_error relative (of the derivative's two terms), with no absolute part, as far as
    the normal density stays a normal fp32 number (|z| < 13.2)."""
    zs = spread(-13.1, 13.1, dt, 8192)
    zs = torch.cat((zs, zs[:-zs.numel() % rows])) if zs.numel() % rows else zs
    w = torch.zeros(8, 8, dtype=dt, device="cuda")
    w[0] = 1.0
    got = []
    for part in zs.view(-1, rows):
        x = torch.zeros(rows, 8, dtype=dt, device="cuda")
        x[:, 0] = part  # one product with 1: the kernel's z is exact
        got.append(cx.linear(x, w, activation="gelu")[:, 5])
    z = zs.double()
    ref = R.value(z, "gelu")
    R.assert_within(torch.cat(got), ref, R.u(dt) * ref.abs() + 1.01 * R.act_error(z, "gelu") * ref.abs() + R.TINY[dt], "value")
    n = zs.numel()
    one = torch.ones(1, n, dtype=dt, device="cuda")
    db = cx.linear_backward(one, one[:, :8], torch.ones(8, n, dtype=dt, device="cuda"), zs[None], activation="gelu",
                            need_dx=False, need_dw=False)[2]
    ref = R.slope(z, "gelu")
    size = 0.5 * torch.special.erfc(-z / math.sqrt(2)) + z.abs() * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    R.assert_within(db, ref, R.u(dt) * ref.abs() + 1.01 * (R.act_error(z, "gelu") + 2.0 ** -22) * size + R.TINY[dt], "slope")


# ------------------------------------------------------------------ matrices side by side in one buffer
def beside(*parts, gap=0):
    """The same matrices as column slices of one buffer (NaN between them)."""
    rows = parts[0].shape[0]
    buf = torch.full((rows, sum(t.shape[1] + gap for t in parts)), float("nan"), dtype=parts[0].dtype, device="cuda")
    out, at = [], 0
    for t in parts:
        v = buf[:, at:at + t.shape[1]]
        v.copy_(t)
        out.append(v)
        at += t.shape[1] + gap
    return buf, out


@pytest.mark.parametrize("m,n,k", [(2, 8, 8), (40, 136, 264), (300, 264, 136), (140, 264, 6208), (1500, 520, 72), (70, 33, 45)])
@pytest.mark.parametrize("gated", [False, True])
def test_forward_between_columns_of_one_buffer(m, n, k, gated):
    g = gen(m)
    wide = 2 * n if gated else n
    x, r, w = rnd(g, m, k), rnd(g, m, n), rnd(g, k, wide, scale=k ** -0.5)
    y, z = torch.zeros_like(r), torch.zeros(m, wide, dtype=BF, device="cuda")
    for gap in (0, 8, 3):
        buf, (xs, ys, rs, zs) = beside(x, y, r, z, gap=gap)
        holes = torch.isnan(buf)
        if gated:
            cx.gated_linear(xs, w, activation="silu", out=ys, preact=zs)
        else:
            cx.linear(xs, w, None, rs, activation="silu", out=ys, preact=zs)
        yr, zr, ey, ez = R.linear(x, w, None, None if gated else r, "silu", False, gated)
        R.assert_within(ys, yr, ey, "y")
        R.assert_within(zs, zr, ez, "z")
        assert torch.equal(torch.isnan(buf), holes) and torch.equal(xs, x) and torch.equal(rs, r)


@pytest.mark.parametrize("rows,cols", [(5, 8), (300, 256), (40, 1001), (9, 4096), (3, 20000)])
@pytest.mark.parametrize("dt", [BF, F32])
def test_norm_and_dropout_between_columns_of_one_buffer(rows, cols, dt):
    g = gen(rows)
    x, w = rnd(g, rows, cols, dtype=dt), rnd(g, cols, dtype=dt)
    for gap in (0, 8):
        buf, (xs, ys) = beside(x, torch.zeros_like(x), gap=gap)
        holes = torch.isnan(buf)
        cx.layer_norm(xs, w, out=ys)
        ref, _, _, bound, _, _ = R.layer_norm(x, w, None, 1e-5)
        R.assert_within(ys, ref, bound)
        cx.dropout(xs, 0.3, 5, 9, out=ys)
        assert torch.equal(ys, cx.dropout(x, 0.3, 5, 9))
        assert torch.equal(torch.isnan(buf), holes) and torch.equal(xs, x)


@pytest.mark.parametrize("gated", [False, True])
def test_backward_between_columns_of_one_buffer(gated):
    """Through the C ABI, which lets a caller place dX: beside dY, X and Z; dW beside W."""
    lib, g = N.lib(), gen(3)
    stream = torch.cuda.current_stream().cuda_stream
    m, n, k = 140, 136, 264
    wide = 2 * n if gated else n
    x, dy, z, w = rnd(g, m, k), rnd(g, m, n), rnd(g, m, wide), rnd(g, k, wide, scale=k ** -0.5)
    buf, (dys, xs, zs, dxs) = beside(dy, x, z, torch.zeros_like(x))
    wbuf, (ws, dws) = beside(w, torch.zeros_like(w))
    db = torch.empty(wide, dtype=BF, device="cuda")
    ld, ldw = buf.stride(0), wbuf.stride(0)
    name = "cuopx_gated_linear_backward" if gated else "cuopx_linear_backward"
    args = (N.BF16, 0, 4, 0, m, n, k, dys.data_ptr(), ld, xs.data_ptr(), ld, ws.data_ptr(), ldw, zs.data_ptr(), ld,
            dxs.data_ptr(), ld, dws.data_ptr(), ldw, db.data_ptr())
    need = getattr(lib, name + "_workspace_size")(L._LINEAR_BACKWARD.pack(*args, 0, 0))
    scratch = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
    assert getattr(lib, name)(L._LINEAR_BACKWARD.pack(*args, scratch.data_ptr() if need else 0, need), stream) == N.SUCCESS
    for what, t, (ref, bound) in zip(("dx", "dw", "db"), (dxs, dws, db), R.linear_backward(dy, x, w, z, "silu", False, gated)):
        R.assert_within(t, ref, bound, what)
    assert torch.equal(dys, dy) and torch.equal(xs, x) and torch.equal(zs, z) and torch.equal(ws, w)


def test_columns_that_do_overlap_are_refused():
    """One shared column, or a slice that runs on into the next row's columns of the other."""
    buf = torch.zeros(40, 64, dtype=BF, device="cuda")
    w = torch.zeros(16, 16, dtype=BF, device="cuda")
    x = buf[:, :16]
    flat = buf.view(-1)
    wrapped = flat[56:56 + 38 * 64].as_strided((38, 16), (64, 1), 56)  # columns 56..63 and 0..7 of the next row
    for call in (lambda: cx.linear(x, w, out=buf[:, 15:31]), lambda: cx.linear(x, w, out=x),
                 lambda: cx.linear(x, w, out=buf[:, 16:32], preact=buf[:, 31:47]),
                 lambda: cx.linear(x, w, residual=buf[:, 16:32], out=buf[:, 17:33]),
                 lambda: cx.linear(x[:38], w, out=wrapped), lambda: cx.linear(x[:20], w, out=buf.view(80, 32)[:20, 16:]),
                 lambda: cx.layer_norm(x, out=buf[:, 15:31]), lambda: cx.layer_norm(x[:38], out=wrapped),
                 lambda: cx.dropout(x, 0.5, 1, out=buf[:, 8:24]), lambda: cx.dropout(x[:38], 0.5, 1, out=wrapped)):
        with pytest.raises(cx.CuopError):
            call()


# ------------------------------------------------------------------ rows that end inside a 16-byte group
def guarded(rows, cols, dt, at=0):
    """A rows x cols matrix whose rows start on 16-byte boundaries and end anywhere, NaN all around it, also right behind
    its last element."""
    ld = (cols + at + 7) // 8 * 8 + 8
    buf = torch.full((8 + rows * ld + 8,), float("nan"), dtype=dt, device="cuda")
    return buf[8:8 + rows * ld].view(rows, ld)[:, at:at + cols], buf


def only_inside(view, buf):
    """Whether every NaN around the matrix is still there and none is left in it."""
    return not torch.isnan(view).any() and int((~torch.isnan(buf)).sum()) == view.numel()


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("m,n,k", [(20, 3, 64), (300, 3, 128), (300, 61, 72), (200, 377, 1024), (140, 70, 6208), (513, 257, 136),
                                   (2600, 1027, 136)])
def test_forward_writes_end_where_rows_end(m, n, k, gated):
    g = gen(n)
    for dt in (BF, HF):
        wide = 2 * n if gated else n
        x, w = rnd(g, m, k, dtype=dt), rnd(g, k, wide, scale=k ** -0.5, dtype=dt)
        (y, ybuf), (z, zbuf) = guarded(m, n, dt), guarded(m, wide, dt)
        if gated:
            cx.gated_linear(x, w, activation="silu", out=y, preact=z)
        else:
            cx.linear(x, w, activation="silu", out=y, preact=z)
        yr, zr, ey, ez = R.linear(x, w, None, None, "silu", False, gated)
        R.assert_within(y, yr, ey, "y")
        R.assert_within(z, zr, ez, "z")
        assert only_inside(y, ybuf) and only_inside(z, zbuf), cx.last_kernel()


# ------------------------------------------------------------------ gradients whose rows end inside one
@pytest.mark.parametrize("trans_w", [0, 1])
@pytest.mark.parametrize("m,n,k", [(20, 133, 77), (300, 61, 135), (1100, 261, 523), (300, 1027, 37)])
def test_backward_writes_end_where_rows_end(m, n, k, trans_w):
    """Through the C ABI, which lets a caller place dX and dW."""
    lib, g = N.lib(), gen(k)
    stream = torch.cuda.current_stream().cuda_stream
    x, dy, z = rnd(g, m, k), rnd(g, m, n), rnd(g, m, n)
    w = rnd(g, *((n, k) if trans_w else (k, n)), scale=k ** -0.5)
    (dx, dxb), (dw, dwb) = guarded(m, k, BF), guarded(*w.shape, BF)
    db = torch.empty(n, dtype=BF, device="cuda")
    args = (N.BF16, trans_w, 4, 0, m, n, k, dy.data_ptr(), n, x.data_ptr(), k, w.data_ptr(), w.shape[1], z.data_ptr(), n,
            dx.data_ptr(), dx.stride(0), dw.data_ptr(), dw.stride(0), db.data_ptr())
    need = lib.cuopx_linear_backward_workspace_size(L._LINEAR_BACKWARD.pack(*args, 0, 0))
    ws = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
    assert lib.cuopx_linear_backward(L._LINEAR_BACKWARD.pack(*args, ws.data_ptr() if need else 0, need), stream) == N.SUCCESS
    for what, t, (ref, bound) in zip(("dx", "dw", "db"), (dx, dw, db), R.linear_backward(dy, x, w, z, "silu", bool(trans_w), False)):
        R.assert_within(t, ref, bound, what)
    assert only_inside(dx, dxb) and only_inside(dw, dwb)


# ------------------------------------------------------------------ documented values
def test_relu_of_special_values():
    """z > 0 ? z : +0, so NaN gives 0, with a derivative of 0."""
    x = torch.zeros(4, 8, dtype=BF, device="cuda")
    x[:, 0] = torch.tensor([INF, -INF, float("nan"), -3.0])
    w = torch.zeros(8, 8, dtype=BF, device="cuda")
    w[0] = 1.0
    y = cx.linear(x, w, activation="relu")
    assert (y[0] == INF).all() and (y[1:] == 0).all() and not torch.signbit(y[1:]).any()
    one = torch.ones(1, 4, dtype=BF, device="cuda")
    z = x[:, 0].contiguous()[None]
    db = cx.linear_backward(one, one, torch.ones(4, 4, dtype=BF, device="cuda"), z, activation="relu",
                            need_dx=False, need_dw=False)[2]
    assert db.tolist() == [1.0, 0.0, 0.0, 0.0]


def test_activations_below_the_normal_range_are_zero():
    """s(z) and the normal density count as 0 where they leave fp32's normal range (z < -87.3, |z| > 13.2)."""
    x = torch.zeros(2, 8, dtype=BF, device="cuda")
    w = torch.zeros(8, 8, dtype=BF, device="cuda")
    w[0] = 1.0
    for act, inside, beyond in (("silu", -86.0, -95.0), ("sigmoid", -86.0, -95.0), ("gelu", -13.0, -14.0)):
        x[0, 0], x[1, 0] = inside, beyond
        y = cx.linear(x, w, activation=act)
        assert (y[0] != 0).all() and (y[1] == 0).all(), act


def test_fp16_dz_beyond_its_range():
    """dZ is rounded to the operands' type for the two products: in fp16 it is infinite beyond 65504 while db, summed from
    the unrounded dZ, is not; in bf16 the same numbers are in range."""
    for dt in (HF, BF):
        dy = torch.full((2, 8), 300.0, dtype=dt, device="cuda")
        z = torch.full((2, 16), 20.0, dtype=dt, device="cuda")
        z[0, 8:], z[1, 8:] = 300.0, -299.0
        x, w = torch.ones(2, 8, dtype=dt, device="cuda"), torch.full((8, 16), 1.0 / 512, dtype=dt, device="cuda")
        dx, dw, db = cx.gated_linear_backward(dy, x, w, z, activation="silu")
        assert torch.isfinite(db).all()
        assert torch.isfinite(dx).all() == (dt == BF)


# ------------------------------------------------------------------ single rows, in-place gradients, repeated calls
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("trans_w", [False, True])
@pytest.mark.parametrize("m,n,k", [(1, 1024, 1200), (1, 2731, 520), (1, 520, 2047), (2, 1032, 1032), (3, 4096, 264)])
def test_single_rows_backward_through_the_tensor_cores(m, n, k, trans_w, gated):
    """2^20 multiplications and more: aligned operands, or copies of unaligned ones; dW has a depth of one to three."""
    g = gen(n)
    wide = 2 * n if gated else n
    for dt, act in ((BF, "silu"), (HF, "gelu")):
        x, dy, z = rnd(g, m, k, dtype=dt), rnd(g, m, n, dtype=dt), rnd(g, m, wide, dtype=dt)
        w = rnd(g, *((wide, k) if trans_w else (k, wide)), scale=k ** -0.5, dtype=dt)
        fn = cx.gated_linear_backward if gated else cx.linear_backward
        got = fn(dy, x, w, z, activation=act, trans_w=trans_w)
        for name, t, (ref, bound) in zip(("dx", "dw", "db"), got, R.linear_backward(dy, x, w, z, act, trans_w, gated)):
            R.assert_within(t, ref, bound, name)


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("rows,cols", [(1, 8), (50, 96), (700, 512), (900, 333), (300, 1001), (400, 4096), (160, 8192),
                                       (40, 16384), (5, 20001), (160, 65536)])
def test_norm_gradient_in_place_of_dy(rows, cols, dt):
    """dX may be dY: the same bits as apart from it."""
    lib, g = N.lib(), gen(cols)
    stream = torch.cuda.current_stream().cuda_stream
    x, dy, w = rnd(g, rows, cols, dtype=dt), rnd(g, rows, cols, dtype=dt), rnd(g, cols, dtype=dt)
    mean, rstd = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    cx.layer_norm(x, w, mean=mean, rstd=rstd)
    ref = cx.layer_norm_backward(dy, x, mean, rstd, w)
    grad, dw, db = dy.clone(), torch.empty_like(w), torch.empty_like(w)
    code = N.F32 if dt == F32 else N.BF16
    args = (code, code, rows, cols, 0.0, x.data_ptr(), cols, w.data_ptr(), 0, 0, 0, mean.data_ptr(), rstd.data_ptr(),
            grad.data_ptr(), cols, grad.data_ptr(), cols, dw.data_ptr(), db.data_ptr())
    need = lib.cuopx_layer_norm_backward_workspace_size(L._NORM.pack(*args, 0, 0))
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    assert lib.cuopx_layer_norm_backward(L._NORM.pack(*args, ws.data_ptr(), need), stream) == N.SUCCESS
    for a, b in zip((grad, dw, db), ref):
        assert torch.equal(a, b)


def test_repeated_calls_give_the_same_bits():
    g = gen(17)
    for m, n, k in ((4, 1024, 1024), (200, 520, 1024), (999, 683, 512), (1500, 1032, 512)):
        x, dy, z = rnd(g, m, k, dtype=HF), rnd(g, m, n, dtype=HF), rnd(g, m, 2 * n, dtype=HF)
        w = rnd(g, k, 2 * n, scale=k ** -0.5, dtype=HF)
        first = (cx.gated_linear(x, w, activation="silu"),) + cx.gated_linear_backward(dy, x, w, z, activation="gelu")
        for _ in range(3):
            again = (cx.gated_linear(x, w, activation="silu"),) + cx.gated_linear_backward(dy, x, w, z, activation="gelu")
            for a, b in zip(first, again):
                assert torch.equal(a, b)
