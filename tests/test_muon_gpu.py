"""Orthogonalised updates on the GPU against the iteration in 64 bits, within
what the kernels' roundings to fp16 predict (muon_refs.py): shapes from one
element to several tiles, stacks, strides and types, streams, graphs, the
optimiser step, and a layer that is trained with it and then served in int8."""
import threading

import pytest
import torch

import cuop_b200 as cx
import int8_refs as Q
import layer_refs as L
import muon_refs as R
from cuop_b200 import _native as N

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
FIVE = [R.COEFFICIENTS] * 5


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def gradient(g, m, n, kind="noise", dtype=F32):
    x = torch.randn(m, n, generator=g, device="cuda")
    if kind == "few":  # a few large directions
        x = 0.05 * x + torch.randn(m, 4, generator=g, device="cuda") @ torch.randn(4, n, generator=g, device="cuda")
    if kind == "decay":  # singular values that fall by a factor of a thousand
        u, s, v = torch.linalg.svd(x, full_matrices=False)
        x = (u * torch.logspace(0, -3, len(s), device="cuda")) @ v
    return (x * 1e-3).to(dtype)


def check(g, coefficients=FIVE, **kw):
    o = cx.orthogonalize(g, steps=len(coefficients), coefficients=coefficients, **kw)
    assert o.shape == g.shape
    for x, y in zip(g.view(-1, *g.shape[-2:]) if g.dim() == 3 else [g], o.view(-1, *g.shape[-2:]) if g.dim() == 3 else [o]):
        x0 = R.normalised(x)
        off = float(torch.linalg.matrix_norm(y.double() - R.iterate(x0, coefficients)))
        assert off <= R.allowed(x0, coefficients, o.dtype), (off, R.predicted(x0, coefficients), cx.last_kernel())
    return o


SHAPES = [(1, 1), (1, 2), (1, 300), (300, 1), (3, 3), (2, 9), (16, 16), (17, 40), (64, 64), (100, 31), (127, 129), (128, 128),
          (129, 127), (200, 333), (256, 256), (257, 300), (300, 257), (64, 1500), (1500, 72), (500, 520), (520, 513), (513, 1100)]


@pytest.mark.parametrize("kind", ["noise", "few", "decay"])
@pytest.mark.parametrize("m,n", SHAPES)
def test_shapes(m, n, kind):
    g = gradient(gen(m + 3 * n), m, n, kind)
    check(g)
    check(g.to(BF))
    check(g.to(HF) * 100, out=torch.empty(m, n, device="cuda"))


@pytest.mark.parametrize("m,n", [(64, 64), (200, 333), (333, 200), (1, 7), (300, 1030), (1030, 300)])
@pytest.mark.parametrize("steps", [0, 1, 2, 3, 8])
def test_steps(m, n, steps):
    check(gradient(gen(steps), m, n, "few"), [R.COEFFICIENTS] * steps)


@pytest.mark.parametrize("m,n", [(200, 333), (520, 300)])
def test_coefficients_of_each_step(m, n):
    """A schedule of its own for every step, cubic steps and ones that grow or shrink among them."""
    for coefficients in ([(1.5, -0.5, 0.0)] * 6, [(3.0, -16 / 5, 6 / 5), (1.875, -1.25, 0.375), R.COEFFICIENTS],
                         [(2.0, 0.0, 0.0), (0.25, 0.0, 0.0)], [(0.0, 1.0, 0.0)], [(8.0, -20.0, 12.0), (1.5, -0.5, 0.0)],
                         [(0.0, 0.0, 0.0)] * 2):
        check(gradient(gen(1), m, n, "noise"), coefficients)


@pytest.mark.parametrize("shape", [(40, 2000), (64, 3001), (3000, 64), (128, 6136), (129, 2500), (300, 5000), (5001, 257), (700, 2600),
                                   (3, 100, 4000), (2, 4000, 200), (20, 70, 1800), (256, 16384)])
def test_long_and_narrow(shape):
    """Several pairs share a tile of the Gram matrix."""
    g = torch.randn(shape, generator=gen(sum(shape)), device="cuda")
    check(g)
    first = cx.orthogonalize(g)
    for _ in range(5):
        assert torch.equal(first, cx.orthogonalize(g))


def test_larger():
    """Several tiles of each kernel, too large for singular values of every step: against the reference norm by norm."""
    for m, n in ((2100, 1030), (1000, 4100), (2560, 2570)):
        g = gradient(gen(m), m, n, "few", BF)
        check(g)


def test_singular_values_and_vectors():
    """U and V stay, singular values follow the polynomial."""
    g = gradient(gen(5), 96, 160, "decay")
    o = check(g, out=torch.empty(96, 160, device="cuda")).double()
    u, s, v = torch.linalg.svd(R.normalised(g), full_matrices=False)
    core = u.mT @ o @ v.mT
    off = core - torch.diag(core.diagonal())
    want = R.iterate(torch.diag(s), FIVE).diagonal()
    bound = R.allowed(R.normalised(g), FIVE, F32)
    assert torch.linalg.matrix_norm(off) <= bound and torch.linalg.vector_norm(core.diagonal() - want) <= bound


@pytest.mark.parametrize("shape", [(3, 64, 64), (5, 100, 260), (2, 300, 140), (9, 17, 33), (4, 520, 513), (1, 70, 90)])
def test_stacks(shape):
    """Each matrix of a stack by itself: the bits of single calls."""
    g = torch.stack([gradient(gen(i), *shape[1:], ["noise", "few"][i % 2]) * 10 ** (i % 5 - 2) for i in range(shape[0])])
    for dt in (BF, F32):
        o = check(g.to(dt))
        for i in range(shape[0]):
            one = cx.orthogonalize(g[i].to(dt))
            assert torch.linalg.matrix_norm((one - o[i]).double()) <= 1e-3 * torch.linalg.matrix_norm(one.double())


def wide(t, left, right, fill):
    """The same stack as column slices of a wider buffer."""
    buf = torch.full((*t.shape[:-1], left + t.shape[-1] + right), fill, dtype=t.dtype, device="cuda")
    v = buf[..., left:left + t.shape[-1]]
    v.copy_(t)
    return v, buf


@pytest.mark.parametrize("shape", [(70, 90), (90, 70), (3, 130, 257), (128, 128), (300, 520)])
@pytest.mark.parametrize("left,right", [(0, 8), (8, 8), (1, 0), (3, 4), (0, 1)])
def test_strides_and_alignment(shape, left, right):
    g0 = torch.randn(shape, generator=gen(7), device="cuda")
    for dt in (BF, F32):
        want = cx.orthogonalize(g0.to(dt))
        g, _ = wide(g0.to(dt), left, right, float("nan"))
        out, buf = wide(torch.zeros_like(g0).to(dt), left, right, 5.0)
        assert torch.equal(cx.orthogonalize(g, out=out), want)
        out.fill_(5.0)
        assert (buf == 5.0).all()
        assert torch.equal(cx.orthogonalize(g, out=g), want)  # in place


def test_matrices_side_by_side():
    """The two projections of a gated weight [K, 2N] as a stack of column slices."""
    w = torch.randn(96, 2 * 130, generator=gen(2), device="cuda")
    halves = w.view(96, 2, 130).transpose(0, 1)
    o = torch.empty(96, 260, device="cuda").view(96, 2, 130).transpose(0, 1)
    cx.orthogonalize(halves, out=o)
    for i in range(2):
        one = cx.orthogonalize(halves[i].contiguous())
        assert (one - o[i]).norm() <= 1e-3 * one.norm()


@pytest.mark.parametrize("dt", [BF, HF, F32])
def test_values(dt):
    """Zeros, the smallest and the largest numbers, and what is not a number."""
    z = torch.zeros(40, 60, dtype=dt, device="cuda")
    assert (cx.orthogonalize(z) == 0).all()
    assert (cx.orthogonalize(z, eps=0.0) != 0).all()  # 0 / 0
    big = torch.full((40, 60), torch.finfo(dt).max, dtype=dt, device="cuda")
    x0 = torch.full((40, 60), 1 / 2400 ** 0.5, dtype=torch.float64, device="cuda")
    ref = R.iterate(x0, FIVE)
    got = cx.orthogonalize(big, out=torch.empty(40, 60, device="cuda"))
    assert (got.double() - ref).norm() <= R.allowed_equal(1.0, FIVE)
    tiny = torch.full((40, 60), torch.finfo(dt).tiny, dtype=dt, device="cuda")
    got = cx.orthogonalize(tiny, eps=0.0, out=torch.empty(40, 60, device="cuda"))
    assert (got.double() - ref).norm() <= R.allowed_equal(1.0, FIVE)
    one = torch.randn(3, 40, 60, device="cuda").to(dt)
    for v in (float("nan"), float("inf")):
        bad = one.clone()
        bad[1, 2, 3] = v
        o = cx.orthogonalize(bad)
        assert torch.isnan(o[1]).all() and torch.equal(o[0], cx.orthogonalize(one)[0]) and torch.isfinite(o[2]).all()


def test_same_bits_every_time():
    for shape in ((100, 260), (1030, 520), (4, 300, 300)):
        g = torch.randn(shape, generator=gen(3), device="cuda").to(BF)
        first = cx.orthogonalize(g)
        for _ in range(10):
            assert torch.equal(first, cx.orthogonalize(g))


def test_streams_threads_and_graphs():
    gs = [torch.randn(s, generator=gen(i), device="cuda") for i, s in enumerate(((300, 520), (1030, 300), (64, 64), (3, 200, 129)))]
    want = [cx.orthogonalize(g) for g in gs]
    streams = [torch.cuda.Stream() for _ in gs]
    torch.cuda.synchronize()
    got = [None] * 4

    def work(i):
        for _ in range(15):
            got[i] = cx.orthogonalize(gs[i], stream=streams[i])

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # two graphs, replayed at the same time
    ins = [gs[0].clone(), gs[1].clone()]
    graphs, outs = [], []
    for i in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(cx.orthogonalize(ins[i]))
        graphs.append(gr)
    for turn in range(4):
        for i in range(2):
            ins[i].copy_(gs[i] * (turn + 1) + turn)
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(outs[i], cx.orthogonalize(gs[i] * (turn + 1) + turn))


def reference_step(w, g, m, lr, mu, decay, nesterov, scale, mdtype):
    m = (mu * m.double() + g.double())
    kept = m.to(mdtype)
    u = g.double() + mu * kept.double() if nesterov else kept.double()
    o = torch.stack([R.iterate(R.normalised(x), FIVE) for x in u.reshape(-1, *u.shape[-2:])]).reshape(u.shape)
    return (1 - lr * decay) * w.double() - lr * scale * o, m, u


@pytest.mark.parametrize("shape", [(60, 90), (200, 130), (2, 100, 257), (520, 300), (1, 40)])
@pytest.mark.parametrize("wt,gt,mt", [(BF, BF, F32), (F32, F32, F32), (BF, F32, BF), (HF, HF, HF), (F32, BF, BF)])
@pytest.mark.parametrize("nesterov", [True, False])
def test_step(shape, wt, gt, mt, nesterov):
    g0 = gen(sum(shape))
    w = (torch.randn(shape, generator=g0, device="cuda") * 0.05).to(wt)
    g = torch.randn(shape, generator=g0, device="cuda").to(gt)
    m = torch.randn(shape, generator=g0, device="cuda").to(mt)
    lr, mu, decay, scale = 0.02, 0.9, 0.1, 0.2 * max(shape[-2:]) ** 0.5
    wr, mr, u = reference_step(w, g, m, lr, mu, decay, nesterov, scale, mt)
    w1, m1 = w.clone(), m.clone()
    assert cx.muon_step(w1, g, m1, lr=lr, mu=mu, weight_decay=decay, nesterov=nesterov) is w1
    # momentum: one fused fp32 operation (mu itself rounded, 2^-24) and its rounding; a kept value next to a border may
    # round the other way, which moves u by one spacing there, far below what the norm allows
    assert ((m1.double() - mr).abs() <= L.u(mt) * mr.abs() + 4 * 2.0 ** -24 * (mu * m.double().abs() + g.double().abs()) + L.TINY[mt]).all()
    for i in range(shape[0] if len(shape) == 3 else 1):
        pick = (lambda t: t[i]) if len(shape) == 3 else (lambda t: t)
        bound = lr * scale * R.allowed(R.normalised(pick(u)), FIVE, F32)
        # u moved where kept values rounded the other way: at most a share of 1e-3 of them
        off = torch.linalg.matrix_norm(pick(w1).double() - pick(wr))
        assert off <= 1.1 * bound + L.u(wt) * torch.linalg.matrix_norm(pick(wr)) + 1e-6 * torch.linalg.matrix_norm(pick(w).double())
    # strided and unaligned operands give the same bits
    w2, wb = wide(w, 3, 2, 9.0)
    m2, mb = wide(m, 1, 0, 9.0)
    cx.muon_step(w2, wide(g, 0, 1, float("nan"))[0], m2, lr=lr, mu=mu, weight_decay=decay, nesterov=nesterov)
    assert torch.equal(w2, w1) and torch.equal(m2, m1)
    w2.fill_(9.0), m2.fill_(9.0)
    assert (wb == 9.0).all() and (mb == 9.0).all()


def test_learning_rate_of_a_graph():
    """lr_tensor multiplies lr, and the decay's share of it, when the kernel runs."""
    w0 = torch.randn(100, 130, generator=gen(1), device="cuda")
    g = torch.randn(100, 130, generator=gen(2), device="cuda")
    w, m = w0.clone(), torch.zeros_like(w0)
    factor = torch.ones(1, device="cuda")
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        cx.muon_step(w, g, m, lr=0.1, weight_decay=0.5, lr_tensor=factor)
    w.copy_(w0), m.zero_()
    ws, ms = w0.clone(), torch.zeros_like(w0)
    for f in (1.0, 0.5, 0.0, 2.0):
        factor.fill_(f)
        gr.replay()
        cx.muon_step(ws, g, ms, lr=0.1 * f, weight_decay=0.5)
        assert torch.equal(m, ms) and (w - ws).abs().max() <= 1e-5 * ws.abs().max()


def test_a_layer_trained_and_served():
    """Steps of a linear layer: forward, gradient, Muon step; then its weight in int8, served."""
    k, n, tokens = 200, 136, 64
    g0 = gen(11)
    w = (torch.randn(k, n, generator=g0, device="cuda") * k ** -0.5).to(BF)
    momentum = torch.zeros(k, n, device="cuda")
    mr = torch.zeros(k, n, dtype=torch.float64, device="cuda")
    for _ in range(3):
        x = torch.randn(tokens, k, generator=g0, device="cuda").to(BF)
        z = torch.empty(tokens, n, dtype=BF, device="cuda")
        y = cx.linear(x, w, activation="silu", preact=z)
        _, dw, _ = cx.linear_backward((2 * y.float() / tokens).to(BF), x, w, z, activation="silu", need_dx=False)
        wr, mr, u = reference_step(w, dw, momentum, 0.02, 0.95, 0.0, True, 0.2 * k ** 0.5, F32)
        cx.muon_step(w, dw, momentum, lr=0.02)
        bound = 0.02 * 0.2 * k ** 0.5 * R.allowed(R.normalised(u), FIVE, F32)
        assert torch.linalg.matrix_norm(w.double() - wr) <= bound + L.u(BF) * torch.linalg.matrix_norm(wr) + 1e-6
    q, s = cx.quantize_int8(w, trans=True)
    qr, sr = Q.quantize(w.t())
    assert torch.equal(q, qr) and torch.equal(s, sr)
    for m in (1, 64, 300):
        x = torch.randn(m, k, generator=g0, device="cuda").to(BF)
        xq, xs = Q.quantize(x)
        y, bound = Q.linear(xq, xs, q, s, None, None, "silu", BF, False)
        L.assert_within(cx.int8_linear(x, q, s, activation="silu"), y, bound, "served")


def test_empty():
    for shape in ((0, 5), (5, 0), (0, 3, 4), (2, 0, 4)):
        g = torch.empty(shape, device="cuda")
        assert cx.orthogonalize(g).shape == shape
        assert cx.muon_step(g, g.clone(), g.clone(), lr=0.1) is g


def test_refusals():
    g = torch.randn(40, 60, device="cuda")
    bad = [
        lambda: cx.orthogonalize(g.cpu()), lambda: cx.orthogonalize(g.double()), lambda: cx.orthogonalize(g[0]),
        lambda: cx.orthogonalize(g.t()), lambda: cx.orthogonalize(g, out=g[:, :59]), lambda: cx.orthogonalize(g, out=g.double()),
        lambda: cx.orthogonalize(g, steps=-1), lambda: cx.orthogonalize(g, steps=33), lambda: cx.orthogonalize(g, eps=-1.0),
        lambda: cx.orthogonalize(g, eps=float("nan")), lambda: cx.orthogonalize(g, coefficients=(1.0, 2.0)),
        lambda: cx.orthogonalize(g, coefficients=[(1.0, 0.0, 0.0)] * 4), lambda: cx.orthogonalize(g, coefficients=3.0),
        lambda: cx.orthogonalize(g, coefficients=(float("inf"), 0.0, 0.0)), lambda: cx.orthogonalize(g, coefficients=(50.0, 0.0, 0.0)),
        lambda: cx.orthogonalize(g[:1].expand(40, 60)), lambda: cx.orthogonalize(g[None].expand(3, 40, 60)),
        lambda: cx.orthogonalize(g, out=g.view(BF).view(40, 120)[:, :60]),
        lambda: cx.orthogonalize(g[:, :30], out=g[:, 30:]),
        lambda: cx.muon_step(g, g, torch.zeros_like(g), lr=0.1), lambda: cx.muon_step(g, torch.zeros_like(g), g, lr=0.1),
        lambda: cx.muon_step(g, torch.zeros_like(g), torch.zeros(40, 61, device="cuda"), lr=0.1),
        lambda: cx.muon_step(g, torch.zeros_like(g), torch.zeros_like(g), lr=float("inf")),
        lambda: cx.muon_step(g, torch.zeros_like(g), torch.zeros_like(g), lr=0.1, lr_tensor=torch.ones(2, device="cuda")),
        lambda: cx.muon_step(g, torch.zeros_like(g), torch.zeros_like(g), lr=0.1, lr_tensor=torch.ones(1)),
        lambda: cx.muon_step(g, torch.zeros_like(g).double(), torch.zeros_like(g), lr=0.1),
    ]
    keep = g.clone()
    for i, call in enumerate(bad):
        with pytest.raises(N.CuopError):
            call()
            print("accepted:", i)
    assert torch.equal(g, keep)
