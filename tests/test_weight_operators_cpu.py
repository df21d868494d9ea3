"""int8 layers and orthogonalised updates without a GPU: refusals before any
launch, workspace sizes, and the definitions that the GPU tests compare with."""
import ctypes as C
import math

import pytest
import torch

import cuop_b200 as cx
import int8_refs as Q
import layer_refs as L
import muon_refs as R
from cuop_b200 import _native as N
from cuop_b200 import int8 as I
from cuop_b200 import muon as M

A = 1 << 32  # far apart addresses, never dereferenced
BAD, TYPE, OK, ROOM = N.INVALID_ARGUMENT, N.UNSUPPORTED_TYPE, N.SUCCESS, N.RESOURCE_UNAVAILABLE
FIVE = (C.c_double * 15)(*(R.COEFFICIENTS * 5))


def quant(**kw):
    v = dict(dtype=N.BF16, trans=0, rows=4, cols=8, X=A, ldx=8, Q=2 * A, ldq=8, scale=3 * A, ws=0, wsb=0)
    v.update(kw)
    return I._QUANTIZE.pack(*v.values())


def lin(**kw):
    v = dict(dtype=N.BF16, act=0, M=4, N=8, K=16, X=A, ldx=16, xs=0, W=2 * A, ldw=16, ws=3 * A, bias=0, R=0, ldr=0, Y=4 * A,
             ldy=8, work=5 * A, wsb=1 << 20)
    v.update(kw)
    return I._INT8.pack(*v.values())


def ortho(**kw):
    v = dict(dtype=N.BF16, out_dtype=N.BF16, steps=5, reserved=0, batch=1, rows=40, cols=60, eps=1e-7, k=C.addressof(FIVE), G=A,
             ldg=60, sg=0, out=2 * A, ldo=60, so=0, ws=3 * A, wsb=1 << 20)
    v.update(kw)
    return M._ORTHO.pack(*v.values())


def muon(**kw):
    v = dict(wd=N.BF16, gd=N.BF16, md=N.F32, steps=5, nesterov=1, reserved=0, batch=1, rows=40, cols=60, eps=1e-7,
             k=C.addressof(FIVE), lr=0.1, mu=0.9, decay=0.0, scale=1.0, lr_dev=0, W=A, ldw=60, sw=0, m=2 * A, ldm=60, sm=0, G=3 * A,
             ldg=60, sg=0, ws=4 * A, wsb=1 << 20)
    v.update(kw)
    return M._MUON.pack(*v.values())


@pytest.mark.parametrize("change,status", [
    (dict(dtype=N.F64), TYPE), (dict(dtype=9), TYPE), (dict(trans=2), BAD), (dict(rows=-1), BAD), (dict(cols=-1), BAD),
    (dict(X=0), BAD), (dict(Q=0), BAD), (dict(scale=0), BAD), (dict(ldx=7), BAD), (dict(ldq=7), BAD), (dict(X=A + 1), BAD),
    (dict(scale=3 * A + 2), BAD), (dict(Q=A), BAD), (dict(Q=A + 62), BAD), (dict(scale=A + 4), BAD), (dict(scale=2 * A + 4), BAD),
    (dict(trans=1, rows=20000, ldq=20000), ROOM), (dict(trans=1, rows=20000, ldq=20000, ws=4 * A, wsb=31), ROOM),
    (dict(trans=1, rows=20000, ldq=19999, ws=4 * A, wsb=32), BAD), (dict(trans=1, ldq=3), BAD),
    (dict(trans=1, rows=20000, ldq=20000, ws=4 * A + 4, wsb=32), BAD), (dict(trans=1, ldq=4, ws=4 * A + 4, wsb=32), BAD),
    (dict(trans=1, rows=20000, ldq=20000, ws=A, wsb=32), BAD), (dict(rows=1 << 31), BAD),
    (dict(rows=1 << 30, ldx=1 << 40), BAD), (dict(trans=1, rows=65535 * 128 + 1, ldq=1 << 24, ws=4 * A, wsb=1 << 20), BAD),
    (dict(rows=0), OK), (dict(trans=1, cols=0), OK)])
def test_quantize_refusals(change, status):
    assert N.lib().cuopx_quantize(quant(**change), None) == status
    assert N.lib().cuopx_quantize(None, None) == BAD


@pytest.mark.parametrize("change,status", [
    (dict(dtype=N.F32), TYPE), (dict(dtype=9), TYPE), (dict(act=6), BAD), (dict(act=-1), BAD), (dict(M=-1), BAD), (dict(N=-1), BAD),
    (dict(K=-1), BAD), (dict(K=131072, ldx=131072, ldw=131072), BAD), (dict(X=0), BAD), (dict(W=0), BAD), (dict(Y=0), BAD),
    (dict(ws=0), BAD), (dict(ldx=15), BAD), (dict(ldw=15), BAD), (dict(ldy=7), BAD), (dict(R=6 * A, ldr=7), BAD),
    (dict(X=A + 1), BAD), (dict(xs=6 * A + 2), BAD), (dict(ws=3 * A + 1), BAD), (dict(bias=6 * A + 1), BAD), (dict(Y=4 * A + 1), BAD),
    (dict(Y=A), BAD), (dict(Y=2 * A + 64), BAD), (dict(Y=3 * A), BAD), (dict(xs=4 * A), BAD), (dict(bias=4 * A + 8), BAD),
    (dict(R=4 * A, ldr=9), BAD), (dict(R=4 * A + 2, ldr=8), BAD), (dict(M=40, work=0), ROOM), (dict(M=40, wsb=64), ROOM),
    (dict(work=5 * A + 8), BAD), (dict(M=40, work=A), BAD), (dict(M=40, work=4 * A), BAD), (dict(M=40, work=3 * A), BAD),
    (dict(M=1 << 40, ldx=1 << 40), BAD), (dict(ldw=1 << 60), BAD), (dict(M=0), OK), (dict(N=0), OK)])
def test_int8_linear_refusals(change, status):
    assert N.lib().cuopx_int8_linear(lin(**change), None) == status
    assert N.lib().cuopx_int8_linear(None, None) == BAD


def test_int8_gated_refusals():
    lib = N.lib()
    assert lib.cuopx_int8_gated_linear(lin(R=6 * A, ldr=8), None) == BAD  # no residual
    assert lib.cuopx_int8_gated_linear(lin(Y=2 * A + 128, ldy=8), None) == BAD  # the second projection's rows of W
    assert lib.cuopx_int8_gated_linear(lin(N=0), None) == OK


def test_int8_workspace():
    lib = N.lib()
    size = lambda **kw: lib.cuopx_int8_linear_workspace_size(lin(**kw))  # noqa: E731
    assert size() == 0  # few enough rows for the product's own kernel
    assert size(M=17) == 512 + 256  # quantised X, scales
    assert size(M=16, K=1024, ldx=1024, ldw=1024) == 16 * 1024 + 256 and size(M=8, K=1024, ldx=1024, ldw=1024) == 0
    assert size(M=1, K=8192, ldx=8192, ldw=8192) == 0 and size(M=1, K=8192, ldx=8192, ldw=8192, N=9000) == 8192 + 256
    assert size(xs=6 * A) == 0
    assert size(M=100, K=100, ldx=100, N=200, ldw=112) == 100 * 112 + 64 + 512  # rounded up to 256 each
    assert size(xs=6 * A, M=100, K=100, ldx=100, N=200, ldw=112) == (100 * 112 + 255) // 256 * 256
    assert size(xs=6 * A, M=100, K=100, ldx=112, N=200, ldw=100) == (200 * 112 + 255) // 256 * 256
    assert lib.cuopx_int8_gated_linear_workspace_size(lin(xs=6 * A, M=100, K=100, ldx=112, N=200, ldw=100)) == 400 * 112
    assert size(xs=6 * A, M=1, K=31, ldx=31, N=8, ldw=31) == 0  # too small to copy for
    assert size(xs=6 * A, M=2, K=65, ldx=65, N=8, ldw=65) == 256 + 768
    assert size(M=0) == 0 and size(K=0) == 0
    # maxima of columns that no cluster holds
    assert lib.cuopx_quantize_workspace_size(quant(trans=1, cols=1000)) == 0
    assert lib.cuopx_quantize_workspace_size(quant(trans=1, rows=12289, cols=1000)) == 4000
    assert lib.cuopx_quantize_workspace_size(quant(trans=0, rows=12289, cols=1000)) == 0


@pytest.mark.parametrize("change,status", [
    (dict(dtype=N.F64), TYPE), (dict(out_dtype=7), TYPE), (dict(steps=-1), BAD), (dict(steps=33), BAD), (dict(reserved=1), BAD),
    (dict(batch=-1), BAD), (dict(rows=-1), BAD), (dict(cols=-1), BAD), (dict(eps=-1.0), BAD), (dict(eps=math.inf), BAD),
    (dict(eps=math.nan), BAD), (dict(k=0), BAD), (dict(G=0), BAD), (dict(out=0), BAD), (dict(ldg=59), BAD), (dict(ldo=59), BAD),
    (dict(G=A + 1), BAD), (dict(out=2 * A + 1), BAD), (dict(out=A + 2), BAD), (dict(out=A, ldo=61), BAD),
    (dict(out=A, out_dtype=N.F16), BAD), (dict(ws=0), ROOM), (dict(wsb=1000), ROOM), (dict(ws=3 * A + 8), BAD), (dict(ws=A), BAD),
    (dict(ws=2 * A), BAD), (dict(batch=2), BAD), (dict(batch=2, sg=2399, so=2400), BAD), (dict(batch=2, sg=59, so=2400), BAD),
    (dict(rows=1 << 25), BAD), (dict(batch=70000), BAD), (dict(ldg=1 << 60), BAD),
    (dict(rows=0), OK), (dict(cols=0), OK), (dict(batch=0), OK)])
def test_orthogonalize_refusals(change, status):
    assert N.lib().cuopx_orthogonalize(ortho(**change), None) == status
    assert N.lib().cuopx_orthogonalize(None, None) == BAD


@pytest.mark.parametrize("triple", [(math.nan, 0, 0), (0, math.inf, 0), (1025.0, 0, 0), (50.0, 0, 0), (0.0, 0.0, 5000.0)])
def test_coefficients_that_run_away(triple):
    """Singular values in [0, 1] that could grow beyond 1024 within five steps."""
    k = (C.c_double * 15)(*(triple * 5))
    assert N.lib().cuopx_orthogonalize(ortho(k=C.addressof(k)), None) == BAD
    assert N.lib().cuopx_muon_step(muon(k=C.addressof(k)), None) == BAD


@pytest.mark.parametrize("change,status", [
    (dict(wd=N.F64), TYPE), (dict(gd=9), TYPE), (dict(md=9), TYPE), (dict(steps=33), BAD), (dict(nesterov=2), BAD),
    (dict(reserved=1), BAD), (dict(lr=math.nan), BAD), (dict(mu=math.inf), BAD), (dict(decay=math.nan), BAD),
    (dict(scale=math.inf), BAD), (dict(eps=-1.0), BAD), (dict(W=0), BAD), (dict(m=0), BAD), (dict(G=0), BAD), (dict(ldw=59), BAD),
    (dict(ldm=59), BAD), (dict(ldg=59), BAD), (dict(W=A + 1), BAD), (dict(m=2 * A + 2), BAD), (dict(lr_dev=5 * A + 1), BAD),
    (dict(G=A), BAD), (dict(G=2 * A), BAD), (dict(W=2 * A), BAD), (dict(lr_dev=A), BAD), (dict(lr_dev=2 * A), BAD),
    (dict(ws=0), ROOM), (dict(wsb=100), ROOM), (dict(ws=4 * A + 128), BAD), (dict(ws=A), BAD), (dict(ws=2 * A), BAD),
    (dict(batch=2), BAD), (dict(batch=2, sw=2400, sm=2400, sg=100), BAD), (dict(rows=0), OK), (dict(cols=0), OK), (dict(batch=0), OK)])
def test_muon_refusals(change, status):
    assert N.lib().cuopx_muon_step(muon(**change), None) == status
    assert N.lib().cuopx_muon_step(None, None) == BAD


def test_python_refuses_without_a_gpu():
    x = torch.zeros(4, 16)
    for call in (lambda: cx.quantize_int8(x), lambda: cx.int8_linear(x.bfloat16(), x.to(torch.int8), x[:, 0]),
                 lambda: cx.int8_gated_linear(x.bfloat16(), x.to(torch.int8), x[:, 0]), lambda: cx.orthogonalize(x),
                 lambda: cx.muon_step(x, x, x, lr=0.1)):
        with pytest.raises(N.CuopError):
            call()


def test_quantize_definition():
    """Half a step off at most; ties to even; rows that are zero, tiny or no numbers."""
    x = torch.randn(20, 33, generator=torch.Generator().manual_seed(0))
    x[3] = 0
    x[4, 5] = math.inf
    x[5, 6] = math.nan
    x[6] *= 1e-35
    x[7, 0], x[7, 1:] = 2.0, 1.0
    q, s = Q.quantize(x)
    rows = [i for i in range(20) if i not in (4, 5)]
    off = (q.double() * s.double()[:, None] - x.double())[rows].abs()
    assert (off <= s.double()[rows, None] / 2 * (1 + 1e-6)).all()
    assert (q[3] == 0).all() and (q[4] == 0).all() and math.isinf(s[4]) and math.isnan(s[5]) and (q[7, 1:] == 64).all()
    assert float(s[6]) >= 2.0 ** -107 and (q[6] == 0).all()


def test_int8_linear_definition():
    g = torch.Generator().manual_seed(1)
    xq = torch.randint(-127, 128, (3, 40), generator=g).to(torch.int8)
    wq = torch.randint(-127, 128, (6, 40), generator=g).to(torch.int8)
    xs, ws, b = torch.rand(3, generator=g), torch.rand(6, generator=g), torch.randn(6, generator=g).bfloat16()
    y, bound = Q.linear(xq, xs, wq, ws, b, None, "none", torch.bfloat16, False)
    for i in range(3):
        for j in range(6):
            z = sum(int(a) * int(c) for a, c in zip(xq[i], wq[j])) * float(xs[i]) * float(ws[j]) + float(b[j])
            assert abs(z - float(y[i, j])) <= 1e-12 * abs(z)
    assert (bound >= L.u(torch.bfloat16) * y.abs()).all()


@pytest.mark.parametrize("shape", [(1, 1), (3, 3), (16, 16), (64, 150), (150, 64), (90, 90)])
@pytest.mark.parametrize("kind", ["noise", "few"])
def test_predicted_errors(shape, kind):
    """The prediction against roundings made in 64 bits: within a factor of two from 16 rows on."""
    g = torch.Generator().manual_seed(sum(shape))
    x = torch.randn(shape, generator=g, dtype=torch.float64)
    if kind == "few":
        x = 0.05 * x + torch.randn(shape[0], 2, generator=g, dtype=torch.float64) @ torch.randn(2, shape[1], generator=g, dtype=torch.float64)
    x0 = R.normalised(x)
    for steps in (1, 3, 5):
        k = [R.COEFFICIENTS] * steps
        off = float((R.rounded_iteration(x0, k) - R.iterate(x0, k)).norm())
        assert off <= R.allowed(x0, k, torch.float64)
        if min(shape) >= 16:
            assert 0.5 * R.predicted(x0, k) <= off <= 2 * R.predicted(x0, k)


def test_iteration_moves_singular_values_only():
    x0 = R.normalised(torch.randn(20, 31, generator=torch.Generator().manual_seed(3)))
    u, s, v = torch.linalg.svd(x0, full_matrices=False)
    for _ in range(5):
        a, b, c = R.COEFFICIENTS
        s = a * s + b * s ** 3 + c * s ** 5
    assert ((u * s) @ v - R.iterate(x0, [R.COEFFICIENTS] * 5)).norm() < 1e-12
    assert (R.iterate(x0, [R.COEFFICIENTS] * 5).mT - R.iterate(x0.mT, [R.COEFFICIENTS] * 5)).norm() < 1e-12
