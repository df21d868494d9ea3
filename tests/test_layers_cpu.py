"""Feed-forward layer operators without a GPU: refusals before any launch,
workspace sizes, the definitions that the GPU tests compare with."""
import subprocess
from pathlib import Path

import pytest
import torch

import cuop_b200 as cx
import layer_refs as R
from cuop_b200 import _native as N
from cuop_b200 import layers as L

ROOT = Path(__file__).resolve().parent.parent
A = 1 << 32  # far apart addresses, never dereferenced


def lin(**kw):
    v = dict(dtype=N.BF16, transW=0, act=0, reserved=0, M=4, N=8, K=16, X=A, ldx=16, W=2 * A, ldw=8, bias=0, R=0, ldr=0,
             Y=3 * A, ldy=8, Z=0, ldz=0, ws=0, wsb=0)
    v.update(kw)
    return L._LINEAR.pack(*v.values())


def lin_bwd(**kw):
    v = dict(dtype=N.BF16, transW=0, act=0, reserved=0, M=4, N=8, K=16, dY=A, lddy=8, X=2 * A, ldx=16, W=3 * A, ldw=8, Z=0,
             ldz=0, dX=4 * A, lddx=16, dW=5 * A, lddw=8, db=6 * A, ws=7 * A, wsb=1 << 20)
    v.update(kw)
    return L._LINEAR_BACKWARD.pack(*v.values())


def norm(**kw):
    v = dict(dtype=N.BF16, wdtype=N.F32, rows=4, cols=8, eps=1e-5, X=A, ldx=8, w=2 * A, b=3 * A, Y=4 * A, ldy=8, mean=5 * A,
             rstd=6 * A, dY=7 * A, lddy=8, dX=8 * A, lddx=8, dw=9 * A, db=10 * A, ws=11 * A, wsb=1 << 20)
    v.update(kw)
    return L._NORM.pack(*v.values())


def drop(**kw):
    v = dict(dtype=N.F32, reserved=0, rows=4, cols=8, p=0.5, seed=1, offset=0, dev=0, X=A, ldx=8, R=0, ldr=0, Y=2 * A, ldy=8)
    v.update(kw)
    return L._DROPOUT.pack(*v.values())


BAD, TYPE, OK, ROOM = N.INVALID_ARGUMENT, N.UNSUPPORTED_TYPE, N.SUCCESS, N.RESOURCE_UNAVAILABLE


@pytest.mark.parametrize("change,status", [
    (dict(dtype=N.F32), TYPE), (dict(dtype=9), TYPE), (dict(act=6), BAD), (dict(act=-1), BAD), (dict(reserved=1), BAD),
    (dict(M=-1), BAD), (dict(N=-1), BAD), (dict(K=-1), BAD), (dict(X=0), BAD), (dict(W=0), BAD), (dict(Y=0), BAD),
    (dict(ldx=15), BAD), (dict(ldw=7), BAD), (dict(ldy=7), BAD), (dict(transW=1, ldw=15), BAD), (dict(R=4 * A, ldr=7), BAD),
    (dict(Z=4 * A, ldz=7), BAD), (dict(Y=A), BAD), (dict(Y=2 * A + 64), BAD), (dict(bias=3 * A + 8), BAD),
    (dict(Z=3 * A + 16, ldz=8), BAD), (dict(Z=A, ldz=8), BAD), (dict(R=3 * A + 2, ldr=8), BAD),
    (dict(R=3 * A, ldr=9), BAD), (dict(X=A + 1), BAD), (dict(W=2 * A + 1), BAD), (dict(Y=3 * A + 1), BAD),
    (dict(bias=4 * A + 1), BAD), (dict(R=4 * A + 1, ldr=8), BAD), (dict(Z=4 * A + 1, ldz=8), BAD), (dict(ws=4 * A + 128, wsb=8), BAD),
    (dict(ws=A, wsb=1 << 20), BAD), (dict(M=1 << 40, ldx=1 << 40), BAD), (dict(ldw=1 << 60), BAD), (dict(M=0), OK), (dict(N=0), OK)])
def test_linear_refusals(change, status):
    assert N.lib().cuopx_linear(lin(**change), None) == status


@pytest.mark.parametrize("change,status", [
    (dict(R=4 * A, ldr=8), BAD), (dict(ldw=15), BAD), (dict(ldw=16, Z=4 * A, ldz=15), BAD), (dict(ldw=16, Y=0), BAD),
    (dict(dtype=N.F64), TYPE), (dict(M=0), OK)])
def test_gated_linear_refusals(change, status):
    assert N.lib().cuopx_gated_linear(lin(**change), None) == status


@pytest.mark.parametrize("change,status", [
    (dict(dtype=N.F64), TYPE), (dict(act=7), BAD), (dict(M=-1), BAD), (dict(dY=0), BAD), (dict(X=0), BAD), (dict(W=0), BAD),
    (dict(act=2), BAD), (dict(act=2, Z=8 * A, ldz=7), BAD), (dict(lddy=7), BAD), (dict(lddx=15), BAD), (dict(lddw=7), BAD),
    (dict(dX=A), BAD), (dict(dW=4 * A), BAD), (dict(db=5 * A), BAD), (dict(dX=3 * A), BAD),
    (dict(act=2, Z=8 * A, ldz=8, wsb=0), ROOM), (dict(act=2, Z=8 * A, ldz=8, ws=8 * A), BAD),
    (dict(dY=A + 1), BAD), (dict(X=2 * A + 1), BAD), (dict(W=3 * A + 1), BAD), (dict(act=2, Z=8 * A + 1, ldz=8), BAD),
    (dict(M=1 << 56), BAD), (dict(lddw=1 << 60), BAD), (dict(dX=4 * A + 1), BAD), (dict(dW=5 * A + 1), BAD), (dict(db=6 * A + 1), BAD), (dict(act=2, Z=8 * A, ldz=8, ws=7 * A + 16), BAD),
    (dict(dX=0, dW=0, db=0), OK)])
def test_linear_backward_refusals(change, status):
    assert N.lib().cuopx_linear_backward(lin_bwd(**change), None) == status


def test_gated_backward_needs_the_pre_activation():
    assert N.lib().cuopx_gated_linear_backward(lin_bwd(ldw=16, lddw=16), None) == BAD
    assert N.lib().cuopx_gated_linear_backward(lin_bwd(ldw=16, lddw=16, Z=8 * A, ldz=15), None) == BAD


@pytest.mark.parametrize("change,status", [
    (dict(dtype=N.F64, wdtype=N.F64), TYPE), (dict(wdtype=N.F16), TYPE), (dict(rows=-1), BAD), (dict(eps=-1.0), BAD),
    (dict(eps=float("nan")), BAD), (dict(eps=float("inf")), BAD), (dict(X=0), BAD), (dict(Y=0), BAD), (dict(ldx=7), BAD),
    (dict(ldy=7), BAD), (dict(Y=A + 16), BAD), (dict(Y=2 * A), BAD), (dict(mean=A), BAD), (dict(rstd=5 * A + 4), BAD),
    (dict(X=A + 1), BAD), (dict(Y=4 * A + 1), BAD), (dict(w=2 * A + 2), BAD), (dict(b=3 * A + 2), BAD), (dict(mean=5 * A + 2), BAD),
    (dict(rstd=6 * A + 1), BAD), (dict(rows=1 << 40, ldx=1 << 40), BAD), (dict(rows=0), OK), (dict(cols=0), OK)])
def test_layer_norm_refusals(change, status):
    assert N.lib().cuopx_layer_norm(norm(**change), None) == status


@pytest.mark.parametrize("change,status", [
    (dict(dtype=N.F64, wdtype=N.F64), TYPE), (dict(X=0), BAD), (dict(dY=0), BAD), (dict(mean=0), BAD), (dict(rstd=0), BAD),
    (dict(lddy=7), BAD), (dict(lddx=7), BAD), (dict(dX=A), BAD), (dict(dX=7 * A + 16), BAD), (dict(dw=10 * A), BAD),
    (dict(ws=0), ROOM), (dict(wsb=4), ROOM), (dict(ws=A), BAD), (dict(ws=11 * A + 64), BAD), (dict(dY=7 * A + 1), BAD),
    (dict(dX=8 * A + 1), BAD), (dict(mean=5 * A + 2), BAD), (dict(w=2 * A + 2), BAD), (dict(dw=9 * A + 2), BAD), (dict(db=10 * A + 1), BAD),
    (dict(dX=0, dw=0, db=0), OK)])
def test_layer_norm_backward_refusals(change, status):
    assert N.lib().cuopx_layer_norm_backward(norm(**change), None) == status


@pytest.mark.parametrize("change,status", [
    (dict(dtype=N.F64), TYPE), (dict(rows=-1), BAD), (dict(p=-0.1), BAD), (dict(p=1.1), BAD), (dict(p=float("nan")), BAD),
    (dict(X=0), BAD), (dict(Y=0), BAD), (dict(ldx=7), BAD), (dict(ldy=7), BAD), (dict(R=3 * A, ldr=7), BAD),
    (dict(Y=A + 4), BAD), (dict(Y=A, ldy=9), BAD), (dict(R=2 * A + 4, ldr=8), BAD), (dict(dev=2 * A + 8), BAD),
    (dict(ldx=1 << 60), BAD), (dict(dev=4 * A + 4), BAD), (dict(X=A + 2), BAD), (dict(Y=2 * A + 2), BAD), (dict(R=3 * A + 2, ldr=8), BAD),
    (dict(rows=1 << 40, cols=1 << 40, ldx=1 << 40, ldy=1 << 40), BAD), (dict(rows=0), OK)])
def test_dropout_refusals(change, status):
    assert N.lib().cuopx_dropout(drop(**change), None) == status


def test_null_argument_structs():
    lib = N.lib()
    for name in ("linear", "gated_linear", "linear_backward", "gated_linear_backward", "layer_norm", "layer_norm_backward",
                 "dropout"):
        assert getattr(lib, "cuopx_" + name)(None, None) == BAD
    for name in ("linear", "gated_linear", "linear_backward", "gated_linear_backward", "layer_norm_backward"):
        assert getattr(lib, f"cuopx_{name}_workspace_size")(None) == 0


def test_struct_formats_match_the_header(tmp_path):
    """Sizes of include/cuopx.h's argument structs, from a C compiler, against the packed formats."""
    names = ("linear", "linear_backward", "layer_norm", "dropout")
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include "cuopx.h"\nint main(void) {' + "".join(
        f'printf("%zu ", sizeof(cuopx_{n}_args));' for n in names) + "return 0; }\n")
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(src), "-o", str(tmp_path / "sizes")], check=True)
    out = subprocess.run([str(tmp_path / "sizes")], capture_output=True, text=True, check=True).stdout
    assert [int(v) for v in out.split()] == [s.size for s in (L._LINEAR, L._LINEAR_BACKWARD, L._NORM, L._DROPOUT)]


def test_cpu_tensors_and_unknown_types_are_refused():
    x = torch.zeros(4, 8, dtype=torch.bfloat16)
    v = torch.zeros(4)
    for call in (lambda: cx.linear(x, x, trans_w=True), lambda: cx.gated_linear(x, x, trans_w=True),
                 lambda: cx.linear_backward(x, x, x), lambda: cx.gated_linear_backward(x, x, x, x),
                 lambda: cx.layer_norm(x), lambda: cx.layer_norm_backward(x, x, v, v), lambda: cx.dropout(x, 0.1, 0),
                 lambda: cx.dropout_backward(x, 0.1, 0)):
        with pytest.raises(cx.CuopError):
            call()


def test_definitions_agree_with_differences():
    """The 64-bit gradients that the GPU tests use, against central differences of
    the 64-bit forward: error h^2 / 6 times a third derivative of size one, plus
    cancellation 2^-52 / h."""
    g = torch.Generator().manual_seed(5)
    h = 1e-5
    z = torch.randn(200, generator=g, dtype=torch.float64) * 2
    z = z[z.abs() > 1e-3]
    for act in R.ACTS:
        num = (R.value(z + h, act) - R.value(z - h, act)) / (2 * h)
        assert (num - R.slope(z, act)).abs().max() < 1e-9, act
        assert R.slope(z, act).abs().max() <= R.SLOPE[act]
    x, dy = (torch.randn(3, 7, generator=g, dtype=torch.float64) for _ in range(2))
    w = torch.randn(7, generator=g, dtype=torch.float64)

    def f(x):
        m = x.mean(1, keepdim=True)
        return ((x - m) / torch.sqrt(((x - m) ** 2).mean(1, keepdim=True) + 1e-5) * w * dy).sum()

    mean = x.mean(1)
    rstd = (((x - mean[:, None]) ** 2).mean(1) + 1e-5) ** -0.5
    hh = (x - mean[:, None]) * rstd[:, None]
    t = dy * w
    dx = rstd[:, None] * (t - t.mean(1, keepdim=True) - hh * (t * hh).mean(1, keepdim=True))
    for i in range(3):
        for j in range(7):
            e = torch.zeros_like(x)
            e[i, j] = h
            assert abs((f(x + e) - f(x - e)) / (2 * h) - dx[i, j]) < 1e-8


def test_philox_known_answers():
    """The published known-answer vectors of Philox4x32-10 for a zero key and counter."""
    assert R.philox_words(4, 0, 0) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
