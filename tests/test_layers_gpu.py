"""Feed-forward layer operators on the GPU against their 64-bit definitions
(layer_refs.py, which also derives the tolerances): sizes from nothing to
several tiles, both weight layouts, strided and unaligned operands, single
tokens, in-place operands, streams, captured graphs, and a whole block run
forward and backward."""
import threading

import pytest
import torch

import cuop_b200 as cx
import layer_refs as R
from cuop_b200 import _native as N
from cuop_b200 import layers as L

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def rnd(gen, *shape, scale=1.0, dtype=BF, off_zero=0.0):
    t = torch.randn(*shape, generator=gen, device="cuda") * scale
    if off_zero:
        t = torch.where(t.abs() < off_zero, torch.full_like(t, off_zero), t)
    return t.to(dtype)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def strided(t, pad, shift):
    """The same matrix inside a larger buffer: rows `pad` elements further apart, base `shift` elements in."""
    rows, cols = t.shape
    buf = torch.full((rows * (cols + pad) + shift + 8,), float("nan"), dtype=t.dtype, device=t.device)
    v = buf[shift:shift + rows * (cols + pad)].view(rows, cols + pad)[:, :cols]
    v.copy_(t)
    return v, buf


def operands(g, m, n, k, dt, trans_w, gated, bias, residual):
    wide = 2 * n if gated else n
    x = rnd(g, m, k, dtype=dt)
    w = rnd(g, *((wide, k) if trans_w else (k, wide)), scale=max(k, 1) ** -0.5, dtype=dt)
    return x, w, rnd(g, wide, scale=0.5, dtype=dt) if bias else None, rnd(g, m, n, dtype=dt) if residual else None


def check_linear(x, w, b, r, act, trans_w, gated, preact=True, **kw):
    m, n = x.shape[0], (w.shape[0] if trans_w else w.shape[1]) // (2 if gated else 1)
    z = torch.full((m, 2 * n if gated else n), float("nan"), dtype=x.dtype, device="cuda") if preact else None
    if gated:
        y = cx.gated_linear(x, w, b, activation=act, trans_w=trans_w, preact=z, **kw)
    else:
        y = cx.linear(x, w, b, r, activation=act, trans_w=trans_w, preact=z, **kw)
    yr, zr, ey, ez = R.linear(x, w, b, r, act, trans_w, gated)
    if act == "relu" and (gated or r is not None):  # either side of 0 may be right within z's error
        pass  # the bound covers it: relu's slope is at most 1
    R.assert_within(y, yr, ey, f"y ({cx.last_kernel()})")
    if preact:
        R.assert_within(z, zr, ez, f"z ({cx.last_kernel()})")
    return y, z


# name, rows, outputs, depth: each reaches the kernel of that name (also through aligned copies).
KERNELS = [("linear_simt", 3, 8, 5), ("linear_split", 1, 264, 512), ("linear_split", 16, 136, 2000), ("linear_split", 30, 520, 320),
           ("linear_split", 64, 1000, 700), ("linear_split", 100, 300, 264), ("linear_split", 5, 7, 40000),
           ("linear_pair_k2", 129, 257, 801), ("linear_pair_k2", 700, 264, 1000), ("linear_pair_k2", 300, 1000, 1536),
           ("linear_pair_k4", 140, 264, 6208), ("linear_pair_k4", 512, 257, 8001), ("linear_tc2_256x256", 300, 520, 264),
           ("linear_tc2_256x256", 2600, 2056, 136)]
GATED_KERNELS = [("gated_linear_simt", 3, 8, 5), ("gated_linear_split", 2, 72, 640), ("gated_linear_split", 50, 200, 1032),
                 ("gated_linear_pair_k2", 129, 130, 801), ("gated_linear_pair_k2", 600, 264, 1000),
                 ("gated_linear_tc2_256x128", 300, 264, 264), ("gated_linear_tc2_256x128", 1500, 1032, 200)]


@pytest.mark.parametrize("trans_w", [False, True])
@pytest.mark.parametrize("name,m,n,k", KERNELS + GATED_KERNELS)
def test_every_forward_kernel(name, m, n, k, trans_w):
    g = gen(m + n)
    gated = name.startswith("gated")
    for dt, pad, shift in ((BF, 0, 0), (HF, 8, 8), (BF, 1, 1)):
        x, w, b, r = operands(g, m, n, k, dt, trans_w, gated, True, not gated)
        if pad:
            x, w = strided(x, pad, shift)[0], strided(w, pad, shift)[0]
        check_linear(x, w, b, r, "gelu_tanh", trans_w, gated)
        # below 2^20 multiplications unaligned operands are not copied but take the SIMT kernel
        small = shift == 1 and m * n * (2 if gated else 1) * k < 1 << 20
        assert cx.last_kernel() == (("gated_linear_simt" if gated else "linear_simt") if small else name)
        y = (cx.gated_linear(x, w) if gated else cx.linear(x, w)) if not trans_w else None
        if y is not None and k < 3000:
            act = "silu" if gated else "none"
            ref, _, bound, _ = R.linear(x, w, None, None, act, False, gated)
            R.assert_within(y, ref, bound, "no bias")


SIZES = [(1, 1, 1), (1, 8, 8), (1, 64, 128), (1, 1000, 72), (2, 7, 31), (3, 40, 200), (5, 128, 64), (8, 264, 136),
         (16, 256, 512), (17, 129, 65), (24, 1024, 328), (33, 64, 1024), (64, 136, 96), (65, 512, 264), (129, 128, 64),
         (130, 72, 1000), (200, 333, 77), (257, 264, 256), (300, 1000, 200), (512, 512, 448), (700, 392, 512)]


@pytest.mark.parametrize("trans_w", [False, True])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_forward_sizes(m, n, k, gated, trans_w):
    g = gen(m * 7 + n * 3 + k)
    for i, (dt, act) in enumerate(((BF, "silu"), (HF, "gelu"))):
        x, w, b, r = operands(g, m, n, k, dt, trans_w, gated, bias=i == 0, residual=not gated and i == 1)
        check_linear(x, w, b, r, act, trans_w, gated, preact=i == 0)
        check_linear(x, w, b, r, act, trans_w, gated, preact=i == 1)


@pytest.mark.parametrize("act", R.ACTS)
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("m,n,k", [(1, 512, 256), (40, 200, 136), (300, 520, 128), (70, 33, 45)])
def test_forward_activations(m, n, k, gated, act):
    g = gen(3)
    for dt in (BF, HF):
        x, w, b, r = operands(g, m, n, k, dt, False, gated, True, not gated)
        check_linear(x, w, b, r, act, False, gated)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("m,n,k", [(1, 264, 512), (13, 136, 320), (150, 264, 128), (400, 320, 192)])
@pytest.mark.parametrize("pad,shift", [(8, 8), (16, 0), (3, 0), (8, 1), (5, 3)])
def test_forward_strides(m, n, k, gated, pad, shift):
    """Operands, results and kept pre-activations inside larger buffers: what lies around them is not touched."""
    g = gen(11)
    for trans_w in (False, True):
        x, w, b, r = operands(g, m, n, k, BF, trans_w, gated, True, not gated)
        xs, ws = strided(x, pad, shift)[0], strided(w, pad, shift)[0]
        rs = strided(r, pad, shift)[0] if r is not None else None
        out, obuf = strided(torch.zeros(m, n, dtype=BF, device="cuda"), pad, shift)
        z, zbuf = strided(torch.zeros(m, 2 * n if gated else n, dtype=BF, device="cuda"), pad, shift)
        before = [torch.isnan(o) for o in (obuf, zbuf)]
        if gated:
            cx.gated_linear(xs, ws, b, activation="gelu_tanh", trans_w=trans_w, out=out, preact=z)
        else:
            cx.linear(xs, ws, b, rs, activation="gelu_tanh", trans_w=trans_w, out=out, preact=z)
        yr, zr, ey, ez = R.linear(x, w, b, r, "gelu_tanh", trans_w, gated)
        R.assert_within(out, yr, ey, "y")
        R.assert_within(z, zr, ez, "z")
        assert torch.equal(torch.isnan(obuf), before[0]) and torch.equal(torch.isnan(zbuf), before[1])


@pytest.mark.parametrize("m,n,k", [(1, 256, 256), (20, 264, 128), (300, 256, 64), (37, 51, 20)])
def test_residual_in_place(m, n, k):
    g = gen(2)
    x, w, b, r = operands(g, m, n, k, BF, False, False, True, True)
    yr, _, ey, _ = R.linear(x, w, b, r, "none", False, False)
    out = cx.linear(x, w, b, r, out=r)
    assert out.data_ptr() == r.data_ptr()
    R.assert_within(out, yr, ey)


@pytest.mark.parametrize("gated", [False, True])
def test_forward_empty_sizes(gated):
    for m, n, k in ((0, 8, 8), (4, 0, 8), (0, 0, 0)):
        x = torch.zeros(m, k, dtype=BF, device="cuda")
        w = torch.zeros(k, 2 * n if gated else n, dtype=BF, device="cuda")
        y = (cx.gated_linear if gated else cx.linear)(x, w)
        assert tuple(y.shape) == (m, n)
    # no products at all: the bias alone
    x, w = torch.zeros(5, 0, dtype=BF, device="cuda"), torch.zeros(0, 16, dtype=BF, device="cuda")
    b = rnd(gen(1), 16)
    check_linear(x, w, b, None, "silu", False, gated)


def test_forward_special_values():
    """Infinities and NaN reach the rows that hold them and no others; large finite values saturate the activations."""
    for m in (3, 150):
        for act in ("silu", "gelu", "gelu_tanh", "sigmoid"):
            x = torch.zeros(m, 64, dtype=BF, device="cuda")
            x[0, 0], x[1, 0], x[2, 0] = 1e30, -1e30, float("nan")
            w = torch.zeros(64, 64, dtype=BF, device="cuda")
            w[0] = 1.0
            y = cx.linear(x, w, activation=act).float()
            top = 1.0 if act == "sigmoid" else x[0, 0].float().item()
            assert (y[0] == top).all() and (y[1] == 0).all() and torch.isnan(y[2]).all(), (act, y[:3, 0])
            assert (y[3:] == (0.5 if act == "sigmoid" else 0.0)).all()


def test_forward_is_deterministic_and_row_independent():
    """The same bits twice; a row's result does not depend on the other rows of the batch."""
    g = gen(9)
    for m, n, k in ((4, 1024, 2048), (48, 512, 1024), (256, 512, 512), (256, 512, 2048), (300, 520, 6400)):
        x, w, b, r = operands(g, m, n, k, BF, False, False, True, True)
        y = cx.linear(x, w, b, r, activation="gelu")
        assert torch.equal(y, cx.linear(x, w, b, r, activation="gelu"))
        x2, r2 = x.clone(), r.clone()
        x2[1:], r2[1:] = float("nan"), 0
        assert torch.equal(y[0], cx.linear(x2, w, b, r2, activation="gelu")[0])


@pytest.mark.parametrize("trans_w", [False, True])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 64, 128), (3, 7, 31), (16, 264, 136), (65, 129, 77), (130, 72, 200),
                                   (257, 264, 256), (300, 1000, 200), (520, 512, 640), (1100, 136, 200),
                                   (300, 1001, 333), (6300, 40, 72)])
def test_backward_sizes(m, n, k, gated, trans_w):
    g = gen(m + n + k)
    for dt, act in ((BF, "silu"), (HF, "gelu"), (BF, "none")):
        if gated and act == "none":
            act = "sigmoid"
        x, w, _, _ = operands(g, m, n, k, dt, trans_w, gated, False, False)
        dy = rnd(g, m, n, dtype=dt)
        z = rnd(g, m, 2 * n if gated else n, dtype=dt, off_zero=1e-3)
        if gated:
            got = cx.gated_linear_backward(dy, x, w, z, activation=act, trans_w=trans_w)
        else:
            got = cx.linear_backward(dy, x, w, z if act != "none" else None, activation=act, trans_w=trans_w)
        for name, t, (ref, bound) in zip(("dx", "dw", "db"), got, R.linear_backward(dy, x, w, z, act, trans_w, gated)):
            R.assert_within(t, ref, bound, f"{name} {act}")


@pytest.mark.parametrize("act", R.ACTS)
@pytest.mark.parametrize("gated", [False, True])
def test_backward_activations(gated, act):
    g = gen(21)
    for m, n, k in ((40, 264, 136), (9, 33, 20)):
        x, w, _, _ = operands(g, m, n, k, HF, False, gated, False, False)
        dy, z = rnd(g, m, n, dtype=HF), rnd(g, m, 2 * n if gated else n, scale=2.0, dtype=HF, off_zero=1e-3)
        fn = cx.gated_linear_backward if gated else cx.linear_backward
        got = fn(dy, x, w, z, activation=act)
        for name, t, (ref, bound) in zip(("dx", "dw", "db"), got, R.linear_backward(dy, x, w, z, act, False, gated)):
            R.assert_within(t, ref, bound, name)
        # any subset of the three gives the same bits
        for need in ((True, False, False), (False, True, False), (False, False, True), (True, False, True)):
            some = fn(dy, x, w, z, activation=act, need_dx=need[0], need_dw=need[1], need_db=need[2])
            for t, full, wanted in zip(some, got, need):
                assert torch.equal(t, full) if wanted else t is None


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("pad,shift", [(8, 8), (3, 0), (8, 1)])
def test_backward_strides(gated, pad, shift):
    g = gen(31)
    for trans_w in (False, True):
        m, n, k = 140, 264, 136
        x, w, _, _ = operands(g, m, n, k, BF, trans_w, gated, False, False)
        dy, z = rnd(g, m, n), rnd(g, m, 2 * n if gated else n)
        fn = cx.gated_linear_backward if gated else cx.linear_backward
        got = fn(*(strided(t, pad, shift)[0] for t in (dy, x, w, z)), activation="gelu", trans_w=trans_w)
        for name, t, (ref, bound) in zip(("dx", "dw", "db"), got, R.linear_backward(dy, x, w, z, "gelu", trans_w, gated)):
            R.assert_within(t, ref, bound, name)


@pytest.mark.parametrize("gated", [False, True])
def test_backward_empty_sizes(gated):
    fn = cx.gated_linear_backward if gated else cx.linear_backward
    t = 2 if gated else 1
    e = lambda *s: torch.zeros(*s, dtype=BF, device="cuda")  # noqa: E731
    dx, dw, db = fn(e(0, 8), e(0, 16), e(16, 8 * t), e(0, 8 * t), activation="silu")  # no rows: sums over nothing
    assert dx.shape == (0, 16) and (dw == 0).all() and (db == 0).all() and dw.shape == (16, 8 * t)
    dx, dw, db = fn(e(4, 0), e(4, 16), e(16, 0), e(4, 0), activation="silu")
    assert dx.shape == (4, 16) and (dx == 0).all() and dw.numel() == 0 and db.numel() == 0
    dx, dw, db = fn(e(4, 8) + 1, e(4, 0), e(0, 8 * t), e(4, 8 * t) + 1, activation="sigmoid")  # no products
    assert dx.numel() == 0 and dw.numel() == 0 and (db != 0).all()


def test_linear_gradient_against_differences():
    """<dx, d> against (f(x + h d) - f(x - h d)) / 2h of the 64-bit forward, f = <dy, y>.  The kernel's dx is off by
    its bound, by what rounding z costs (CURVE u |z|), and the difference by h^2 times a third derivative."""
    g = gen(77)
    m, n, k, act = 6, 40, 24, "gelu"
    for gated in (False, True):
        x, w, b, _ = operands(g, m, n, k, BF, False, gated, True, False)
        dy = rnd(g, m, n)
        z = torch.empty(m, 2 * n if gated else n, dtype=BF, device="cuda")
        if gated:
            cx.gated_linear(x, w, b, activation=act, preact=z)
            dx, dw, db = cx.gated_linear_backward(dy, x, w, z, activation=act)
        else:
            cx.linear(x, w, b, activation=act, preact=z)
            dx, dw, db = cx.linear_backward(dy, x, w, z, activation=act)

        def f(x, w, b):
            zz = x @ w + b
            v = R.value(zz[:, :n], act)
            return (dy.double() * (v * zz[:, n:] if gated else v)).sum()

        X, W, B = x.double(), w.double(), b.double()
        Z, h = X @ W + B, 1e-4
        rel = R.u(BF) * Z.abs() * 1.01  # change of z by its rounding
        if gated:
            a, u, ra, ru = Z[:, :n], Z[:, n:], rel[:, :n], rel[:, n:]
            moved = torch.cat((R.CURVE[act] * ra * u.abs() + R.SLOPE[act] * ru, R.SLOPE[act] * ra), 1)
            moved = moved * torch.cat((dy, dy), 1).double().abs()
        else:
            moved = dy.double().abs() * R.CURVE[act] * rel
        ref = R.linear_backward(dy, x, w, z, act, False, gated)
        for got, d, (_, bound), extra in (
                (dx, torch.randn_like(X), ref[0], moved @ W.abs().t()),
                (dw, torch.randn_like(W), ref[1], X.abs().t() @ moved), (db, torch.randn_like(B), ref[2], moved.sum(0))):
            dirs = [torch.zeros_like(t) for t in (X, W, B)]
            dirs[0 if got is dx else 1 if got is dw else 2] = d
            num = (f(*(t + h * e for t, e in zip((X, W, B), dirs))) - f(*(t - h * e for t, e in zip((X, W, B), dirs)))) / (2 * h)
            allowed = ((bound + extra) * d.abs()).sum() + 1e-4 * (dy.double().abs().sum() + 1)
            assert (num - (got.double() * d).sum()).abs() <= allowed


# ------------------------------------------------------------------ layer norm
NORM_TYPES = [(BF, BF), (BF, F32), (HF, HF), (HF, F32), (F32, F32)]


@pytest.mark.parametrize("dt,wt", NORM_TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 2), (1, 8), (7, 31), (5, 64), (2, 256), (9, 1000), (33, 1001), (1, 4096),
                                       (300, 136), (40, 2048), (17, 5120), (6, 8192), (5, 16384), (3, 20000), (2, 65537)])
def test_layer_norm_sizes(rows, cols, dt, wt):
    g = gen(rows + cols)
    x = rnd(g, rows, cols, scale=2.0, dtype=dt) + 1
    dy = rnd(g, rows, cols, dtype=dt)
    w, b = rnd(g, cols, dtype=wt), rnd(g, cols, dtype=wt)
    mean, rstd = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    y = cx.layer_norm(x, w, b, mean=mean, rstd=rstd)
    yr, mr, rr, ey, em, er = R.layer_norm(x, w, b, 1e-5)
    R.assert_within(y, yr, ey, "y")
    R.assert_within(mean, mr, em, "mean")
    R.assert_within(rstd, rr, er, "rstd")
    assert torch.equal(y, cx.layer_norm(x, w, b))
    got = cx.layer_norm_backward(dy, x, mean, rstd, w)
    for name, t, (ref, bound) in zip(("dx", "dw", "db"), got, R.layer_norm_backward(dy, x, mean, rstd, w)):
        R.assert_within(t, ref, bound, name)
    for need in ((True, False, False), (False, True, True), (False, False, True), (False, True, False)):
        some = cx.layer_norm_backward(dy, x, mean, rstd, w, need_dx=need[0], need_dw=need[1], need_db=need[2])
        for name, t, (ref, bound), wanted in zip(("dx", "dw", "db"), some, R.layer_norm_backward(dy, x, mean, rstd, w), need):
            assert (t is not None) == wanted
            if wanted:
                R.assert_within(t, ref, bound, name)


@pytest.mark.parametrize("rows,cols", [(5, 40), (700, 512), (1500, 1024), (2003, 96), (1201, 4096), (700, 8192), (301, 16384),
                                       (1500, 333)])
def test_layer_norm_without_weight_or_bias_and_many_rows(rows, cols):
    g = gen(4)
    x, dy = rnd(g, rows, cols), rnd(g, rows, cols)
    mean, rstd = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    w, b = rnd(g, cols), rnd(g, cols)
    for ww, bb in ((None, None), (w, None), (None, b)):
        yr, _, _, ey, _, _ = R.layer_norm(x, ww, bb, 1e-3)
        R.assert_within(cx.layer_norm(x, ww, bb, eps=1e-3, mean=mean, rstd=rstd), yr, ey)
        got = cx.layer_norm_backward(dy, x, mean, rstd, ww)
        for name, t, (ref, bound) in zip(("dx", "dw", "db"), got, R.layer_norm_backward(dy, x, mean, rstd, ww)):
            R.assert_within(t, ref, bound, name)


@pytest.mark.parametrize("pad,shift", [(8, 8), (3, 0), (4, 1)])
@pytest.mark.parametrize("cols", [256, 1000, 77])
def test_layer_norm_strides_and_in_place(cols, pad, shift):
    g = gen(6)
    for dt in (BF, F32):
        x, dy, w, b = rnd(g, 37, cols, dtype=dt), rnd(g, 37, cols, dtype=dt), rnd(g, cols, dtype=dt), rnd(g, cols, dtype=dt)
        yr, _, _, ey, _, _ = R.layer_norm(x, w, b, 1e-5)
        mean, rstd = torch.empty(37, device="cuda"), torch.empty(37, device="cuda")
        xs, xbuf = strided(x, pad, shift)
        out, obuf = strided(torch.zeros_like(x), pad, shift)
        holes = torch.isnan(obuf)
        cx.layer_norm(xs, w, b, out=out, mean=mean, rstd=rstd)
        R.assert_within(out, yr, ey)
        assert torch.equal(torch.isnan(obuf), holes)
        got = cx.layer_norm_backward(strided(dy, pad, shift)[0], xs, mean, rstd, w)
        for name, t, (ref, bound) in zip(("dx", "dw", "db"), got, R.layer_norm_backward(dy, x, mean, rstd, w)):
            R.assert_within(t, ref, bound, name)
        cx.layer_norm(xs, w, b, out=xs)
        R.assert_within(xs, yr, ey)
        assert torch.equal(torch.isnan(xbuf), holes)


def test_layer_norm_constant_rows_large_means_and_empty():
    for dt in (BF, F32):
        x = torch.full((4, 512), 3.0, dtype=dt, device="cuda")  # variance 0
        mean, rstd = torch.empty(4, device="cuda"), torch.empty(4, device="cuda")
        assert (cx.layer_norm(x, mean=mean, rstd=rstd) == 0).all() and (mean == 3).all()
        assert ((rstd - 1e-5 ** -0.5).abs() <= 1e-5 ** -0.5 * 2.0 ** -22).all()
    # a mean a thousand times the spread: summing squares in fp32 would lose the variance
    x = (1000 + torch.randn(8, 1024, generator=gen(1), device="cuda"))
    yr, _, _, ey, _, _ = R.layer_norm(x, None, None, 1e-5)
    R.assert_within(cx.layer_norm(x), yr, ey)
    for shape in ((0, 16), (4, 0)):
        e = torch.zeros(shape, dtype=BF, device="cuda")
        s = torch.zeros(shape[0], device="cuda")
        assert cx.layer_norm(e).shape == shape
        dx, dw, db = cx.layer_norm_backward(e, e, s, s)
        assert dx.shape == shape and (dw == 0).all() and (db == 0).all()


# ------------------------------------------------------------------ dropout
@pytest.mark.parametrize("dt", [BF, HF, F32])
@pytest.mark.parametrize("shape", [(1,), (3,), (4, 5), (1, 64), (7, 33), (16, 128), (129, 1001), (2, 3, 8)])
def test_dropout_values(shape, dt):
    g = gen(8)
    x, r = rnd(g, *shape, dtype=dt), rnd(g, *shape, dtype=dt)
    for p, seed, offset in ((0.5, 0, 0), (0.1, 2 ** 63 + 12345, 2 ** 32 - 3), (0.9, -5, 2 ** 64 - 2)):
        words = torch.tensor(R.philox_words(x.numel(), seed % 2 ** 64, offset), device="cuda", dtype=torch.int64)
        keep = (words >= round(p * 2 ** 32)).view(shape)
        for res in (None, r):
            y = cx.dropout(x, p, seed, offset, residual=res)
            ref = torch.where(keep, x.double() / (1 - p), torch.zeros(1, device="cuda", dtype=torch.float64))
            err = 2.0 ** -23 * ref.abs()  # 1 / (1 - p) and the product in fp32
            if res is not None:
                ref = ref + res.double()
                err = err + 2.0 ** -24 * ref.abs()
            R.assert_within(y, ref, R.u(dt) * ref.abs() + (1 + R.u(dt)) * err + R.TINY[dt])
        dropped = cx.dropout(x, p, seed, offset)
        assert torch.equal(dropped, cx.dropout_backward(x, p, seed, offset))


def test_dropout_edges():
    x = rnd(gen(1), 64, 96)
    assert torch.equal(cx.dropout(x, 0.0, 3), x)
    assert (cx.dropout(x, 1.0, 3) == 0).all()
    assert torch.equal(cx.dropout(x, 1.0, 3, residual=x), x)
    bad = torch.full((4096,), float("nan"), dtype=BF, device="cuda")
    y = cx.dropout(bad, 0.5, 7)  # a dropped NaN or infinity is 0, not NaN
    kept = torch.isnan(y)
    assert (y[~kept] == 0).all() and 1500 < int(kept.sum()) < 2600
    assert cx.dropout(x[:0], 0.5, 1).shape == (0, 96)
    # any split of a tensor at a multiple of four gives the same mask
    whole = cx.dropout(x, 0.3, 11, 100)
    parts = torch.cat((cx.dropout(x[:10], 0.3, 11, 100), cx.dropout(x[10:], 0.3, 11, 100 + 10 * 96 // 4)))
    assert torch.equal(whole, parts)


@pytest.mark.parametrize("cols,pad,shift", [(128, 8, 0), (128, 8, 8), (96, 3, 1), (30, 2, 0), (33, 8, 0)])
def test_dropout_strides_and_in_place(cols, pad, shift):
    g = gen(12)
    x, r = rnd(g, 19, cols), rnd(g, 19, cols)
    ref = cx.dropout(x, 0.4, 99, 7, residual=r)
    xs, rs = strided(x, pad, shift)[0], strided(r, pad, shift)[0]
    out, buf = strided(torch.zeros_like(x), pad, shift)
    holes = torch.isnan(buf)
    assert torch.equal(cx.dropout(xs, 0.4, 99, 7, residual=rs, out=out), ref)
    assert torch.equal(torch.isnan(buf), holes)
    assert torch.equal(cx.dropout(xs, 0.4, 99, 7, residual=r), ref)
    assert torch.equal(cx.dropout(x, 0.4, 99, 7, residual=r, out=r), ref)
    assert torch.equal(cx.dropout(x, 0.4, 99, 7, residual=rs, out=x), ref)


# ------------------------------------------------------------------ refusals of the Python front end
def test_refusals():
    x = torch.zeros(4, 64, dtype=BF, device="cuda")
    w = torch.zeros(64, 32, dtype=BF, device="cuda")
    v = torch.zeros(32, dtype=BF, device="cuda")
    s = torch.zeros(4, device="cuda")
    for call in (
            lambda: cx.linear(x, w[:32]), lambda: cx.linear(x, w.half()), lambda: cx.linear(x.float(), w.float()),
            lambda: cx.linear(x, w, v[:16]), lambda: cx.linear(x, w, v.float()), lambda: cx.linear(x, w, activation="tanh"),
            lambda: cx.linear(x, w, residual=x), lambda: cx.linear(x, w.cpu()), lambda: cx.linear(x[0], w),
            lambda: cx.linear(x[:1].expand(4, 64), w), lambda: cx.linear(x[:, ::2], w[:32]), lambda: cx.linear(x, w, out=x),
            lambda: cx.linear(x, w, out=x[:, :32]), lambda: cx.linear(x, w, preact=x),
            lambda: cx.gated_linear(x, w[:, :31]), lambda: cx.gated_linear(x, w, v[:16]),
            lambda: cx.linear_backward(x, x, w), lambda: cx.linear_backward(x[:, :32], x, w, activation="gelu"),
            lambda: cx.linear_backward(x[:, :1].expand(4, 32), x, w),
            lambda: cx.gated_linear_backward(x[:, :16], x, w, x[:, :31]),
            lambda: cx.layer_norm(x, v), lambda: cx.layer_norm(x.double()), lambda: cx.layer_norm(x, eps=-1.0),
            lambda: cx.layer_norm(x, mean=s[:3]), lambda: cx.layer_norm(x, mean=s, rstd=s),
            lambda: cx.layer_norm(x, s.new_zeros(64).half()), lambda: cx.layer_norm_backward(x, x, s, v),
            lambda: cx.dropout(x, 1.5, 0), lambda: cx.dropout(x, 0.5, 0, residual=w), lambda: cx.dropout(x.double(), 0.5, 0),
            lambda: cx.dropout(x[:, ::2], 0.5, 0), lambda: cx.dropout(x, 0.5, 0, offset_tensor=s)):
        with pytest.raises(cx.CuopError):
            call()


# ------------------------------------------------------------------ streams and graphs
def test_other_stream_and_two_at_once():
    """Calls on two streams at once, with their own scratch, give what they give alone."""
    g = gen(40)
    m, n, k = 200, 264, 328
    x, w, b, r = operands(g, m, n, k, BF, False, False, True, True)
    z = rnd(g, m, n)
    ref = cx.linear(x, w, b, r, activation="gelu")
    refb = cx.linear_backward(r, x, w, z, activation="gelu")
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(20):
        y = cx.linear(x, w, b, r, activation="gelu", stream=s1)
        g1 = cx.linear_backward(r, x, w, z, activation="gelu", stream=s1)
        g2 = cx.linear_backward(r, x, w, z, activation="gelu", stream=s2)
        h = cx.layer_norm(x, stream=s2.cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(y, ref) and torch.equal(h, cx.layer_norm(x))
    for a, b2, c in zip(refb, g1, g2):
        assert torch.equal(a, b2) and torch.equal(a, c)


def test_two_captured_graphs():
    """Two graphs captured one after the other and replayed in turn and together, on new inputs; dropout draws a new
    mask at each replay through offset_tensor."""
    g = gen(41)
    m, n, k = 96, 520, 264
    x, w, b, r = operands(g, m, n, k, BF, True, False, True, True)
    z = rnd(g, m, n)
    mean, rstd = torch.empty(m, device="cuda"), torch.empty(m, device="cuda")
    counter = torch.zeros(1, dtype=torch.int64, device="cuda")

    def step():
        y = cx.linear(x, w, b, r, activation="silu", trans_w=True)
        d = cx.dropout(y, 0.5, 3, offset_tensor=counter)
        counter.add_((m * n + 3) // 4)
        h = cx.layer_norm(d, mean=mean, rstd=rstd)
        return (y, d, h) + cx.linear_backward(r, x, w, z, activation="silu", trans_w=True) + cx.layer_norm_backward(
            r, d, mean, rstd)

    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=s):
            out = step()
        graphs.append((gr, out))
    for i in range(4):
        x.copy_(rnd(g, m, k))
        counter.fill_(1000 * i)
        gr, out = graphs[i % 2]
        gr.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        counter.fill_(1000 * i)
        for t, ref in zip(got, step()):
            assert torch.equal(t, ref)
    first = [t.clone() for t in graphs[0][1]]
    graphs[0][0].replay()
    assert not torch.equal(first[1], graphs[0][1][1])  # the counter moved on


def test_several_host_threads():
    """Four threads with a stream each give what one gives alone."""
    g = gen(43)
    x, w, b, _ = operands(g, 256, 512, 2048, BF, False, False, True, False)
    dy = rnd(g, 256, 512)

    def calls():
        return (cx.linear(x, w, b, activation="gelu"), cx.linear(x[:3], w, b), cx.layer_norm(x)) + cx.linear_backward(dy, x, w)

    ref, bad = calls(), []
    torch.cuda.synchronize()

    def work():
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(10):
                got = calls()
            s.synchronize()
        bad.extend(i for i, (a, c) in enumerate(zip(got, ref)) if not torch.equal(a, c))

    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


@pytest.mark.parametrize("m", [64, 700])
def test_chains_of_dependent_launches(m):
    """Every launch reads what the one before it wrote; launches may start early, their reads may not."""
    g = gen(44)
    x, ws = rnd(g, m, 1024), [rnd(g, 1024, 1024, scale=1 / 32) for _ in range(8)]

    def chain():
        t = x
        for i, w in enumerate(ws):
            t = cx.dropout(cx.layer_norm(cx.linear(t, w, residual=t, activation="silu")), 0.1, i)
        return t

    ref = chain()
    torch.cuda.synchronize()
    t = x
    for i, w in enumerate(ws):  # step by step, each finished before the next
        y = cx.linear(t, w, residual=t, activation="silu")
        torch.cuda.synchronize()
        h = cx.layer_norm(y)
        torch.cuda.synchronize()
        t = cx.dropout(h, 0.1, i)
        torch.cuda.synchronize()
    assert torch.equal(ref, t)
    for _ in range(20):
        assert torch.equal(chain(), ref)


# ------------------------------------------------------------------ workspaces, through the C ABI
def test_workspaces_are_large_enough():
    """Calls with exactly the bytes that the size calls ask for write nothing behind them."""
    lib, g = N.lib(), gen(45)
    stream = torch.cuda.current_stream().cuda_stream
    for m, n, k in ((5, 301, 999), (200, 133, 701), (333, 520, 64)):
        for gated in (0, 1):
            wide = 2 * n if gated else n
            x, w, dy, z = rnd(g, m, k), rnd(g, k, wide, scale=k ** -0.5), rnd(g, m, n), rnd(g, m, wide)
            y, dx, dw, db = (torch.empty_like(t) for t in (dy, x, w, w[0]))
            head = (N.BF16, 0, 4, 0, m, n, k)
            fwd = head + (x.data_ptr(), k, w.data_ptr(), wide, 0, 0, 0, y.data_ptr(), n, 0, 0)
            bwd = head + (dy.data_ptr(), n, x.data_ptr(), k, w.data_ptr(), wide, z.data_ptr(), wide, dx.data_ptr(), k,
                          dw.data_ptr(), wide, db.data_ptr())
            for name, fmt, args in (("linear", L._LINEAR, fwd), ("linear_backward", L._LINEAR_BACKWARD, bwd)):
                name = ("gated_" if gated else "") + name
                need = getattr(lib, f"cuopx_{name}_workspace_size")(fmt.pack(*args, 0, 0))
                ws = torch.full((need + 4096,), 0x5A, dtype=torch.uint8, device="cuda")
                assert getattr(lib, "cuopx_" + name)(fmt.pack(*args, ws.data_ptr() if need else 0, need), stream) == N.SUCCESS
                assert (ws[need:] == 0x5A).all()
            yr, _, ey, _ = R.linear(x, w, None, None, "silu", False, bool(gated))
            R.assert_within(y, yr, ey)
            for t, (ref, bound) in zip((dx, dw, db), R.linear_backward(dy, x, w, z, "silu", False, bool(gated))):
                R.assert_within(t, ref, bound)
            # without a workspace a kernel for any alignment takes the forward call
            y.zero_()
            assert getattr(lib, "cuopx_gated_linear" if gated else "cuopx_linear")(L._LINEAR.pack(*fwd, 0, 0), stream) == 0
            R.assert_within(y, yr, ey)
    for rows, cols in ((7, 96), (900, 1000), (300, 9000), (40, 333)):
        x, dy, w = rnd(g, rows, cols), rnd(g, rows, cols), rnd(g, cols)
        mean, rstd = torch.zeros(rows, device="cuda"), torch.ones(rows, device="cuda")
        dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(w)
        args = (N.BF16, N.BF16, rows, cols, 0.0, x.data_ptr(), cols, w.data_ptr(), 0, 0, 0, mean.data_ptr(), rstd.data_ptr(),
                dy.data_ptr(), cols, dx.data_ptr(), cols, dw.data_ptr(), db.data_ptr())
        need = lib.cuopx_layer_norm_backward_workspace_size(L._NORM.pack(*args, 0, 0))
        ws = torch.full((need + 4096,), 0x5A, dtype=torch.uint8, device="cuda")
        assert lib.cuopx_layer_norm_backward(L._NORM.pack(*args, ws.data_ptr(), need), stream) == N.SUCCESS
        assert (ws[need:] == 0x5A).all()
        for t, (ref, bound) in zip((dx, dw, db), R.layer_norm_backward(dy, x, mean, rstd, w)):
            R.assert_within(t, ref, bound)


# ------------------------------------------------------------------ offsets past 32 bits
def test_rows_past_32_bits():
    """Operands whose last row starts beyond 2^32 bytes (and 2^31 elements)."""
    g = gen(50)
    m, k, n, ld = 3, 64, 128, (1 << 30) + 8 * 1024
    big = torch.zeros(2 * ld + 4096, dtype=BF, device="cuda")

    def far(cols, at):
        return big.as_strided((m, cols), (ld, 1), at)

    x, w, b, r = operands(g, m, n, k, BF, False, False, True, True)
    xs, ys, zs, rs = far(k, 0), far(n, 512), far(n, 1024), far(n, 2048)
    xs.copy_(x)
    rs.copy_(r)
    # interleaved in one buffer: the spans overlap, which the library refuses, so inputs and outputs go one at a time
    yr, zr, ey, ez = R.linear(x, w, b, r, "gelu", False, False)
    R.assert_within(cx.linear(xs, w, b, rs, activation="gelu"), yr, ey)
    z = torch.empty(m, n, dtype=BF, device="cuda")
    cx.linear(x, w, b, r, activation="gelu", out=ys, preact=z)
    R.assert_within(ys, yr, ey)
    cx.linear(x, w, b, r, activation="gelu", preact=zs)
    R.assert_within(zs, zr, ez)
    yr, _, _, ey, _, _ = R.layer_norm(x, None, None, 1e-5)
    R.assert_within(cx.layer_norm(xs), yr, ey)
    assert torch.equal(cx.dropout(xs, 0.5, 1), cx.dropout(x, 0.5, 1))


def test_many_elements():
    """More than 2^31 elements in one call (bf16, 4 GiB a tensor)."""
    rows, cols = (1 << 18) + 1, 8192
    x = torch.zeros(rows, cols, dtype=BF, device="cuda")
    x[-1] = rnd(gen(3), cols)
    y = cx.dropout(x, 0.5, 5)
    last = cx.dropout(x[-1:], 0.5, 5, (rows - 1) * cols // 4)
    assert torch.equal(y[-1:], last) and int((last != 0).sum()) > 3000
    del y
    h = cx.layer_norm(x)
    assert torch.equal(h[-1:], cx.layer_norm(x[-1:]))


# ------------------------------------------------------------------ a whole block
@pytest.mark.parametrize("m,d,f", [(1, 64, 128), (50, 136, 264), (260, 256, 512)])
def test_feed_forward_block(m, d, f):
    """y = x + dropout(gated(norm(x)) W2 + b2) forward and backward, against the same block in 64 bits with the same
    mask.  Each stage rounds its result to bf16 once (2^-8 or less, relative), and the block chains at most eight of
    them, each with derivatives of order one: the relative error of the whole, as a norm, stays under 8 * 2^-8."""
    g = gen(60)
    x = rnd(g, m, d)
    nw, nb = 1 + rnd(g, d, scale=0.1), rnd(g, d, scale=0.1)
    w1, b1 = rnd(g, d, 2 * f, scale=d ** -0.5), rnd(g, 2 * f, scale=0.1)
    w2, b2 = rnd(g, f, d, scale=f ** -0.5), rnd(g, d, scale=0.1)
    dy = rnd(g, m, d)
    p, seed = 0.2, 42
    mean, rstd = torch.empty(m, device="cuda"), torch.empty(m, device="cuda")
    z = torch.empty(m, 2 * f, dtype=BF, device="cuda")
    h = cx.layer_norm(x, nw, nb, mean=mean, rstd=rstd)
    a = cx.gated_linear(h, w1, b1, preact=z)
    y = cx.dropout(cx.linear(a, w2, b2), p, seed, residual=x)
    do = cx.dropout_backward(dy, p, seed)
    da, dw2, db2 = cx.linear_backward(do, a, w2)
    dh, dw1, db1 = cx.gated_linear_backward(da, h, w1, z)
    dxn, dnw, dnb = cx.layer_norm_backward(dh, x, mean, rstd, nw)
    dx = dxn.float() + dy.float()

    leaves = [t.double().requires_grad_() for t in (x, nw, nb, w1, b1, w2, b2)]
    X, NW, NB, W1, B1, W2, B2 = leaves
    H = torch.nn.functional.layer_norm(X, (d,), NW, NB, 1e-5)
    ZZ = H @ W1 + B1
    O = (torch.nn.functional.silu(ZZ[:, :f]) * ZZ[:, f:]) @ W2 + B2
    keep = cx.dropout(torch.ones(m, d, device="cuda"), p, seed) != 0
    Y = X + torch.where(keep, O / (1 - p), torch.zeros_like(O))
    Y.backward(dy.double())
    for name, got, ref in zip(("y", "dx", "dnw", "dnb", "dw1", "db1", "dw2", "db2"),
                              (y, dx, dnw, dnb, dw1, db1, dw2, db2), [Y.detach()] + [t.grad for t in leaves]):
        rel = ((got.double() - ref).norm() / ref.norm()).item()
        assert rel < 8 * 2.0 ** -8, (name, rel)
