"""Orthogonalised updates with operands of 22 bits: float32 results as near the iteration in 64 bits as fp32 sums
allow (muon22_refs.py), more bits or fewer where a caller asks for them."""
import pytest
import torch

import cuop_b200 as cx
import layer_refs as L
import muon22_refs as W
import muon_refs as R
from cuop_b200 import _native as N
from test_muon_gpu import gen, gradient, reference_step, wide

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
FIVE = [R.COEFFICIENTS] * 5


def check(g, coefficients=FIVE, **kw):
    o = cx.orthogonalize(g, steps=len(coefficients), coefficients=coefficients, **kw)
    for x, y in zip(g.reshape(-1, *g.shape[-2:]), o.reshape(-1, *g.shape[-2:])):
        x0 = R.normalised(x)
        off = float(torch.linalg.matrix_norm(y.double() - R.iterate(x0, coefficients)))
        assert off <= W.allowed22(x0, coefficients, o.dtype), (off, W.predicted22(x0, coefficients))
    return o


SHAPES = [(1, 1), (1, 300), (300, 1), (3, 3), (2, 9), (16, 16), (17, 40), (64, 64), (100, 31), (127, 129), (129, 127), (128, 128),
          (200, 333), (256, 256), (257, 300), (300, 257), (500, 520), (520, 513), (513, 1100), (1030, 700)]


@pytest.mark.parametrize("kind", ["noise", "few", "decay"])
@pytest.mark.parametrize("m,n", SHAPES)
def test_float32_results(m, n, kind):
    g = gradient(gen(m + 3 * n), m, n, kind)
    check(g)
    check(g.to(BF), out=torch.empty(m, n, device="cuda"))
    check(g.to(HF) * 100)
    check(g.to(BF), operand_bits=22)


@pytest.mark.parametrize("shape", [(40, 2000), (128, 6136), (3000, 64), (256, 16384), (300, 5000), (5001, 257), (3, 100, 4000), (20, 70, 1800)])
def test_long_and_narrow(shape):
    """Several pairs share a tile of the Gram matrix."""
    g = torch.randn(shape, generator=gen(sum(shape)), device="cuda")
    first = check(g)
    for _ in range(5):
        assert torch.equal(first, cx.orthogonalize(g))


def test_larger():
    for m, n in ((2100, 1030), (1000, 2100)):
        check(gradient(gen(m), m, n, "few", F32))


@pytest.mark.parametrize("m,n", [(64, 64), (200, 333), (333, 200), (300, 1030)])
@pytest.mark.parametrize("steps", [0, 1, 2, 3, 8])
def test_steps(m, n, steps):
    check(gradient(gen(steps), m, n, "few"), [R.COEFFICIENTS] * steps)


def test_coefficients_of_each_step():
    for coefficients in ([(1.5, -0.5, 0.0)] * 6, [(3.0, -16 / 5, 6 / 5), (1.875, -1.25, 0.375), R.COEFFICIENTS],
                         [(2.0, 0.0, 0.0), (0.25, 0.0, 0.0)], [(0.0, 1.0, 0.0)], [(8.0, -20.0, 12.0), (1.5, -0.5, 0.0)],
                         [(0.0, 0.0, 0.0)] * 2):
        check(gradient(gen(1), 200, 333, "noise"), coefficients)


@pytest.mark.parametrize("shape", [(64, 64), (333, 200), (3, 130, 257), (300, 5000)])
def test_bits_as_asked_for(shape):
    """The bits decide, not the result's type: 16-bit results are the float32 ones, rounded."""
    g = torch.randn(shape, generator=gen(1), device="cuda")
    full, fast = cx.orthogonalize(g), cx.orthogonalize(g, operand_bits=11)
    assert torch.equal(full, cx.orthogonalize(g, operand_bits=22)) and not torch.equal(full, fast)
    for dt in (BF, HF):
        out = torch.empty(shape, dtype=dt, device="cuda")
        assert torch.equal(cx.orthogonalize(g, out=out), (fast if dt == BF else full).to(dt))
        assert torch.equal(cx.orthogonalize(g, out=out, operand_bits=11), fast.to(dt))
        assert torch.equal(cx.orthogonalize(g, out=out, operand_bits=22), full.to(dt))
    w, m = torch.randn(shape, generator=gen(2), device="cuda"), torch.zeros(shape, device="cuda")
    for v in (w, w.to(HF), w.to(BF)):
        got = [cx.muon_step(v.clone(), g, m.clone(), lr=0.5, operand_bits=bits) for bits in (None, 11, 22)]
        assert torch.equal(got[0], got[1 if v.dtype == BF else 2]) and not torch.equal(got[1], got[2])
    for bits in (0, 12, 23, -11, "22", True):
        with pytest.raises(N.CuopError):
            cx.orthogonalize(g, operand_bits=bits)
        with pytest.raises(N.CuopError):
            cx.muon_step(w, g, m, lr=0.5, operand_bits=bits)


@pytest.mark.parametrize("shape", [(60, 90), (200, 130), (2, 100, 257), (520, 300)])
@pytest.mark.parametrize("gt,mt", [(F32, F32), (BF, F32), (BF, BF)])
@pytest.mark.parametrize("nesterov", [True, False])
def test_step_of_float32_weights(shape, gt, mt, nesterov):
    g0 = gen(sum(shape))
    w = torch.randn(shape, generator=g0, device="cuda") * 0.05
    g = torch.randn(shape, generator=g0, device="cuda").to(gt)
    m = torch.randn(shape, generator=g0, device="cuda").to(mt)
    lr, mu, decay, scale = 0.02, 0.9, 0.1, 0.2 * max(shape[-2:]) ** 0.5
    kept = cx_momentum(g, m, mu, mt)
    # from the momentum as stored: its own rounding is the business of another test
    u = torch.addcmul(g.double(), kept.double(), torch.tensor(mu, device="cuda").double()) if nesterov else kept.double()
    w1, m1 = w.clone(), m.clone()
    cx.muon_step(w1, g, m1, lr=lr, mu=mu, weight_decay=decay, nesterov=nesterov)
    assert torch.equal(m1, kept)
    for i in range(shape[0] if len(shape) == 3 else 1):
        pick = (lambda t: t[i]) if len(shape) == 3 else (lambda t: t)
        x0 = R.normalised(pick(u))
        wr = (1 - lr * decay) * pick(w).double() - lr * scale * R.iterate(x0, FIVE)
        # u itself is rounded to fp32 when X is made of it, as is mu (2^-24 of it, twice): the iteration carries that
        # along as it does X's own rounding, which allowed22 counts; the weight's two products and its sum, 2^-24 each
        off = torch.linalg.matrix_norm(pick(w1).double() - wr)
        assert off <= lr * scale * 1.1 * W.allowed22(x0, FIVE, F32) + 4 * 2.0 ** -24 * torch.linalg.matrix_norm(pick(w).double())


def cx_momentum(g, m, mu, mt):
    """The momentum as the kernel stores it: one fused operation in fp32 (exact in 64 bits up to its one rounding)."""
    mu32 = torch.tensor(mu, device="cuda").double()
    return (mu32 * m.double() + g.double()).float().to(mt)


@pytest.mark.parametrize("shape", [(70, 90), (90, 70), (3, 130, 257), (300, 520)])
@pytest.mark.parametrize("left,right", [(0, 8), (1, 0), (3, 4)])
def test_strides_and_in_place(shape, left, right):
    g0 = torch.randn(shape, generator=gen(7), device="cuda")
    want = cx.orthogonalize(g0)
    g, _ = wide(g0, left, right, float("nan"))
    out, buf = wide(torch.zeros_like(g0), left, right, 5.0)
    assert torch.equal(cx.orthogonalize(g, out=out), want)
    out.fill_(5.0)
    assert (buf == 5.0).all()
    assert torch.equal(cx.orthogonalize(g, out=g), want)


def test_values():
    z = torch.zeros(40, 60, device="cuda")
    assert (cx.orthogonalize(z) == 0).all() and torch.isnan(cx.orthogonalize(z, eps=0.0)).all()
    one = torch.randn(3, 40, 60, device="cuda")
    for v in (float("nan"), float("inf")):
        bad = one.clone()
        bad[1, 2, 3] = v
        o = cx.orthogonalize(bad)
        assert torch.isnan(o[1]).all() and torch.equal(o[0], cx.orthogonalize(one)[0]) and torch.isfinite(o[2]).all()


def test_two_graphs_at_once():
    gs = [torch.randn(s, generator=gen(i), device="cuda") for i, s in enumerate(((300, 520), (1030, 300)))]
    ins = [g.clone() for g in gs]
    graphs, outs = [], []
    for x in ins:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(cx.orthogonalize(x))
        graphs.append(gr)
    streams = [torch.cuda.Stream() for _ in gs]
    for turn in range(4):
        for x, g in zip(ins, gs):
            x.copy_(g * (turn + 1) + turn)
        torch.cuda.synchronize()
        for gr, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                gr.replay()
        torch.cuda.synchronize()
        for o, g in zip(outs, gs):
            assert torch.equal(o, cx.orthogonalize(g * (turn + 1) + turn))
