"""Operators on a linear layer's weight after its gradient, as they are measured: the
orthogonalised update that trains it, and the 8-bit integer form that serves it.

own is False: run() computes the plain form from elementary torch operations in 32 bits
(64 for the integer sums), rounded once at the end.  own is True: run() calls the operators
of cuop_b200.
"""
import math

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"f16": 2, "bf16": 2, "f32": 4}
ACTS = ("none", "relu", "gelu", "gelu_tanh", "silu", "sigmoid")
COEFFICIENTS = (3.4445, -4.7750, 2.0315)  # of the quintic iteration, five steps
EPS = 1e-7
MU, DECAY = 0.95, 0.01


def listed():
    return [
        # Activations of a prompt batch, one scale a token: what precedes every integer product of a prompt.
        {"name": "quantise rows", "op": "quantize", "m": 8192, "k": 8192, "dtype": "bf16", "trans": False},
        # An odd weight stored [K][N], one scale a column, laid out once for serving as [N][K].
        {"name": "quantise weight odd", "op": "quantize", "m": 4095, "k": 10001, "dtype": "f16", "trans": True},
        # One new token through a small projection with a skip connection: launch latency.
        {"name": "int8 one token", "op": "int8", "m": 1, "k": 1024, "n": 1024, "dtype": "bf16", "act": "none",
         "bias": True, "residual": True, "given": False},
        # A serving batch of 24 single tokens: the weights' bytes count, half of the 16-bit layer's.
        {"name": "int8 24 tokens", "op": "int8", "m": 24, "k": 8192, "n": 8192, "dtype": "bf16", "act": "gelu",
         "bias": True, "residual": False, "given": False},
        # A ragged batch of prompts with a skip connection.
        {"name": "int8 ragged f16", "op": "int8", "m": 1777, "k": 4096, "n": 5000, "dtype": "f16", "act": "gelu_tanh",
         "bias": True, "residual": True, "given": False},
        # Single tokens of four sequences through a gated block's first half.
        {"name": "int8 gated 4 tokens", "op": "int8_gated", "m": 4, "k": 4096, "n": 8192, "dtype": "bf16",
         "act": "silu", "bias": False, "given": False},
        # A prompt batch through it, the activations quantised already (they feed another layer too).
        {"name": "int8 gated prompts", "op": "int8_gated", "m": 8192, "k": 4096, "n": 10240, "dtype": "bf16",
         "act": "silu", "bias": False, "given": True},
        # The gradient of one square projection, the smallest that a model of some size has: latency.
        {"name": "orthogonalise 1024", "op": "ortho", "batch": 1, "m": 1024, "n": 1024, "dtype": "bf16"},
        # A tall and an odd one, from fp32 sums of gradients kept in 16 bits.
        {"name": "orthogonalise tall odd", "op": "ortho", "batch": 1, "m": 5001, "n": 1777, "dtype": "f16"},
        # A whole step for the square projections of eight layers, stacked.
        {"name": "muon stacked", "op": "muon", "batch": 8, "m": 2048, "n": 2048, "dtype": "bf16", "grad": "bf16",
         "nesterov": True},
        # A whole step for the projection between, with gradients summed in fp32.
        {"name": "muon 4096 x 10240", "op": "muon", "batch": 1, "m": 4096, "n": 10240, "dtype": "bf16", "grad": "f32",
         "nesterov": False},
        # The widest weight of the benchmark (8192 x 28672).
        {"name": "muon wide", "op": "muon", "batch": 1, "m": 8192, "n": 28672, "dtype": "bf16", "grad": "bf16",
         "nesterov": True},
    ]


def _size(rng, lo, hi):
    """A length spread over the logarithm of [lo, hi]: round ones, multiples of 8, any."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    step = rng.choice((64, 64, 8, 1))
    return max(lo, min(hi, v // step * step if v >= step else v))


def draw(rng):
    op = rng.choice(("quantize", "int8", "int8", "int8_gated", "ortho", "ortho", "muon", "muon"))
    if op == "quantize":
        while True:
            c = {"op": op, "m": _size(rng, 1, 32768), "k": _size(rng, 16, 16384),
                 "dtype": rng.choice(("bf16", "f16", "f32")), "trans": rng.random() < 0.4}
            if c["m"] * c["k"] <= 8192 * 8192:
                return c
    if op.startswith("int8"):
        while True:
            c = {"op": op, "m": _size(rng, 1, 8192), "k": _size(rng, 64, 16384), "n": _size(rng, 64, 16384),
                 "dtype": rng.choice(("bf16", "bf16", "f16")), "act": rng.choice(ACTS if op == "int8" else ACTS[1:]),
                 "bias": rng.random() < 0.5, "given": rng.random() < 0.3}
            if work(c)["flops"] <= 1.37e12 and (rng.random() < 0.2 or c["m"] * c["k"] * c["n"] > 1 << 24):
                break
        if op == "int8":
            c["residual"] = rng.random() < 0.5
        return c
    while True:
        c = {"op": op, "batch": rng.choice((1, 1, 1, 2, 3, 8)), "m": _size(rng, 64, 8192), "n": _size(rng, 64, 16384),
             "dtype": rng.choice(("bf16", "bf16", "f16"))}
        if rng.random() < 0.5:
            c["m"], c["n"] = c["n"], c["m"]
        if op == "muon":
            c["grad"] = rng.choice((c["dtype"], "f32"))
            c["nesterov"] = rng.random() < 0.5
        if work(c)["flops"] <= 3e13 and (rng.random() < 0.3 or c["m"] * c["n"] > 1 << 18):
            return c


def work(case):
    op, es = case["op"], SIZE[case["dtype"]]
    if op == "quantize":
        m, k = case["m"], case["k"]
        return {"bytes": m * k * (es + 1) + 4 * (k if case["trans"] else m), "flops": 3.0 * m * k}
    if op.startswith("int8"):
        m, k, n = case["m"], case["k"], case["n"]
        wide = 2 * n if op == "int8_gated" else n
        x = m * k + 4 * m if case["given"] else es * m * k
        out = es * m * n * (2 if case.get("residual") else 1)
        return {"bytes": x + wide * (k + 4) + out + (es * wide if case["bias"] else 0), "flops": 2.0 * m * k * wide}
    b, p, q = case["batch"], min(case["m"], case["n"]), max(case["m"], case["n"])
    # a step: X X^T and A A are symmetric, half of their products are needed; B X is whole
    flops = 5.0 * b * (p * p * q + p * p * p + 2.0 * p * p * q)
    if op == "ortho":
        return {"bytes": 2 * es * b * p * q, "flops": flops}
    # gradient in, momentum and weight in and out
    return {"bytes": b * p * q * (SIZE[case["grad"]] + 8 + 2 * es), "flops": flops}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, op = DTYPES[case["dtype"]], case["op"]

    def normal(*shape, scale=1.0, to=dt):
        return (torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * scale).to(to)

    s = {"case": case}
    if op == "quantize" or op.startswith("int8"):
        m, k = case["m"], case["k"]
        x = torch.randn(m, k, generator=g, device="cuda")
        x[:, :: max(1, k // 4 + 1)] *= 12.0  # a few channels are far larger than the others
        if op == "quantize":
            s["x"] = (x * k ** -0.5 if case["trans"] else x).to(dt)
            return s
        wide = 2 * case["n"] if op == "int8_gated" else case["n"]
        # the weights, quantised once and laid out [N][K]; a channel's largest is about four deviations
        s["wq"] = (torch.randn(wide, k, generator=g, device="cuda") * 32).round().clamp(-127, 127).to(torch.int8)
        s["ws"] = (1 + 0.25 * torch.rand(wide, generator=g, device="cuda")) * (k ** -0.5 / 32)
        if k % 16:  # rows on 16-byte boundaries, as the layout for serving has them
            rows = torch.zeros(wide, (k + 15) // 16 * 16, dtype=torch.int8, device="cuda")
            rows[:, :k] = s["wq"]
            s["wq"] = rows[:, :k]
        if case["given"]:
            top = x.abs().amax(1).clamp_min(2.0 ** -100)
            s["x"] = torch.round(x * (127.0 / top)[:, None]).to(torch.int8)
            s["xs"] = top / 127.0
        else:
            s["x"] = x.to(dt)
        if case["bias"]:
            s["bias"] = normal(wide, scale=0.3)
        if case.get("residual"):
            s["residual"] = normal(m, case["n"])
        return s
    b, m, n = case["batch"], case["m"], case["n"]
    shape = (b, m, n) if b > 1 else (m, n)

    def gradient():
        # a few directions that all tokens share, over the noise of the others
        few = torch.randn(b, m, 8, generator=g, device="cuda") * torch.arange(1, 9, device="cuda") ** -0.5
        few = few @ torch.randn(b, 8, n, generator=g, device="cuda")
        return ((few + torch.randn(b, m, n, generator=g, device="cuda")) * 1e-3).view(shape)

    if op == "ortho":
        s["g"] = gradient().to(dt)
        return s
    s["g"] = gradient().to(DTYPES[case["grad"]])
    s["buf"] = gradient() * 8
    s["w"] = normal(*shape, scale=0.02)
    s["lr"] = 0.02
    return s


# ------------------------------------------------------------------ the plain forms
def _act(z, act):
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "sigmoid":
        return 1 / (1 + torch.exp(-z))
    return z


def _quantize(x):
    """Rows of whole numbers from -127 to 127 and the step of each row; a row's largest
    magnitude counts as 2^-100 at least."""
    x = x.float()
    top = x.abs().amax(1).clamp_min(2.0 ** -100)
    most = torch.full_like(top, 127.0)  # a tensor: torch divides by and into Python numbers with another rounding
    return torch.round(x * (most / top)[:, None]), top / most


def _newton_schulz(x):
    """x [batch, m, n] in fp32; singular values towards 1."""
    a, b, c = COEFFICIENTS
    x = x / (torch.sqrt((x.double() * x.double()).sum((1, 2), keepdim=True)) + EPS).float()
    tall = x.shape[1] > x.shape[2]
    if tall:
        x = x.mT
    for _ in range(5):
        gram = x @ x.mT
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.mT if tall else x


def _plain(s):
    c = s["case"]
    op, dt = c["op"], DTYPES[c["dtype"]]
    if op == "quantize":
        q, scale = _quantize(s["x"].t() if c["trans"] else s["x"])
        return [q.to(torch.int8), scale]
    if op.startswith("int8"):
        q, xs = (s["x"], s["xs"]) if c["given"] else _quantize(s["x"])
        # sums of up to 16384 products of up to 127 * 127: beyond 24 bits
        z = (q.double() @ s["wq"].double().t()).float() * xs[:, None] * s["ws"]
        if "bias" in s:
            z = z + s["bias"].float()
        n = c["n"]
        y = _act(z, c["act"]) if op == "int8" else _act(z[:, :n], c["act"]) * z[:, n:]
        if "residual" in s:
            y = y + s["residual"].float()
        return [y.to(dt)]
    g = s["g"].float().view(c["batch"], c["m"], c["n"])
    if op == "ortho":
        return [_newton_schulz(g).to(dt).view(s["g"].shape)]
    buf = MU * s["buf"].view(g.shape) + g
    o = _newton_schulz(g + MU * buf if c["nesterov"] else buf)
    s["buf"].copy_(buf.view(s["buf"].shape))
    w = s["w"].float().view(g.shape)
    w = w * (1 - s["lr"] * DECAY) - s["lr"] * 0.2 * math.sqrt(max(c["m"], c["n"])) * o
    s["w"].copy_(w.view(s["w"].shape))
    return [s["w"], s["buf"]]


# ------------------------------------------------------------------ the framework's calls
def _own(s):
    import cuop_b200 as cx

    c = s["case"]
    op = c["op"]
    if op == "quantize":
        return list(cx.quantize_int8(s["x"], trans=c["trans"]))
    if op == "int8":
        return [cx.int8_linear(s["x"], s["wq"], s["ws"], s.get("bias"), s.get("residual"), x_scale=s.get("xs"),
                               activation=c["act"], dtype=DTYPES[c["dtype"]])]
    if op == "int8_gated":
        return [cx.int8_gated_linear(s["x"], s["wq"], s["ws"], s.get("bias"), x_scale=s.get("xs"),
                                     activation=c["act"], dtype=DTYPES[c["dtype"]])]
    if op == "ortho":
        return [cx.orthogonalize(s["g"], coefficients=COEFFICIENTS, steps=5, eps=EPS)]
    w = cx.muon_step(s["w"], s["g"], s["buf"], lr=s["lr"], mu=MU, weight_decay=DECAY, nesterov=c["nesterov"],
                     coefficients=COEFFICIENTS, steps=5, eps=EPS)
    return [w, s["buf"]]


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------ the definitions in 64 bits
def _value(z, act):
    if act == "relu":
        return z.clamp_min(0)
    if act == "gelu":
        return z * 0.5 * torch.special.erfc(-z / math.sqrt(2.0))
    half = {"none": None, "sigmoid": z, "silu": z}.get(act, 2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
    if half is None:
        return z
    sig = 0.5 * (torch.tanh(0.5 * half) + 1)
    return sig if act == "sigmoid" else z * sig


def _polar(x):
    """The same iteration on the smaller Gram matrix's side, one matrix at a time."""
    out = []
    for m in x.unbind(0):
        m = m / (torch.linalg.vector_norm(m) + EPS)
        left = m.shape[0] <= m.shape[1]
        eye = torch.eye(min(m.shape), dtype=m.dtype, device=m.device)
        for _ in range(5):
            t = torch.mm(m, m.mT) if left else torch.mm(m.mT, m)
            poly = COEFFICIENTS[0] * eye + torch.mm(COEFFICIENTS[1] * eye + COEFFICIENTS[2] * t, t)
            m = torch.mm(poly, m) if left else torch.mm(m, poly)
        out.append(m)
    return torch.stack(out)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    d = {k: v.double() for k, v in s.items() if isinstance(v, torch.Tensor)}
    if op == "quantize":  # whole numbers are defined by fp32 operations: they have no 64-bit value
        return [None, torch.maximum(d["x"].abs().max(0 if case["trans"] else 1)[0], d["x"].new_tensor(2.0 ** -100)) / 127]
    if op.startswith("int8"):
        x = d["x"]
        if not case["given"]:
            x32 = s["x"].float()
            top = torch.linalg.vector_norm(x32, float("inf"), dim=1, keepdim=True).clamp(min=2.0 ** -100)
            x = torch.round(torch.mul(x32, torch.div(torch.tensor(127.0, device="cuda"), top))).double() * (top.double() / 127)
        else:
            x = x * d["xs"][:, None]
        z = torch.mm(x, (d["wq"] * d["ws"][:, None]).mT) + d.get("bias", 0)
        if op == "int8_gated":
            gate, up = z.chunk(2, dim=1)
            return [_value(gate, case["act"]) * up]
        return [_value(z, case["act"]) + d.get("residual", 0)]
    if work(case)["flops"] > 2e13 and case["batch"] > 1:
        return None
    g = d["g"].reshape(case["batch"], case["m"], case["n"])
    if op == "ortho":
        return [_polar(g).reshape(d["g"].shape)]
    buf = torch.add(g, d["buf"].reshape(g.shape), alpha=MU)
    o = _polar(torch.add(g, buf, alpha=MU) if case["nesterov"] else buf).reshape(d["w"].shape)
    step = s["lr"] * 0.2 * max(case["m"], case["n"]) ** 0.5
    return [torch.add((1 - s["lr"] * DECAY) * d["w"], o, alpha=-step), buf.reshape(d["buf"].shape)]
