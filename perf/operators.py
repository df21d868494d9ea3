"""Feed-forward block operators, as they are measured: linear with a fused epilogue, gated
linear, layer norm and dropout, forward and backward.

own is False: run() computes the plain form from elementary torch operations in 32 bits,
rounded once at the end.  own is True: run() calls the operators of cuop_b200.
"""
import math

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"f16": 2, "bf16": 2, "f32": 4}
ACTS = ("none", "relu", "gelu", "gelu_tanh", "silu", "sigmoid")


def listed():
    return [
        # One new token through a small projection with a skip connection: launch latency.
        {"name": "linear one token", "op": "linear", "m": 1, "k": 1024, "n": 1024, "dtype": "bf16", "trans_w": False,
         "act": "none", "bias": True, "residual": True, "preact": False},
        # A serving batch of 24 single tokens, weights stored [N][K]: the weights' bytes count.
        {"name": "linear 24 tokens", "op": "linear", "m": 24, "k": 8192, "n": 8192, "dtype": "bf16", "trans_w": True,
         "act": "gelu", "bias": True, "residual": False, "preact": False},
        # The forward pass of a training step on a ragged batch, which keeps the pre-activation.
        {"name": "linear ragged f16", "op": "linear", "m": 1777, "k": 4096, "n": 5000, "dtype": "f16",
         "trans_w": False, "act": "gelu_tanh", "bias": True, "residual": True, "preact": True},
        # The backward pass of the benchmark's wide bf16 layer (4096 x 8192 by 8192 x 28672).
        {"name": "linear backward wide", "op": "linear_backward", "m": 4096, "k": 8192, "n": 28672, "dtype": "bf16",
         "trans_w": False, "act": "gelu"},
        # Single tokens of four sequences through a gated block's first half.
        {"name": "gated 4 tokens", "op": "gated", "m": 4, "k": 4096, "n": 8192, "dtype": "bf16", "trans_w": False,
         "act": "silu", "bias": False, "preact": False},
        # A training batch through it, which keeps both pre-activations.
        {"name": "gated training", "op": "gated", "m": 8192, "k": 4096, "n": 10240, "dtype": "bf16", "trans_w": True,
         "act": "silu", "bias": False, "preact": True},
        # Its backward pass on a ragged batch and an odd width.
        {"name": "gated backward odd", "op": "gated_backward", "m": 999, "k": 2048, "n": 2731, "dtype": "f16",
         "trans_w": True, "act": "gelu"},
        # The norm before a projection for a few single tokens: launch latency.
        {"name": "norm 8 tokens", "op": "norm", "m": 8, "n": 8192, "dtype": "bf16", "stats": False},
        # The norm over a ragged fp32 batch, with the statistics that the backward pass takes.
        {"name": "norm ragged f32", "op": "norm", "m": 20011, "n": 1000, "dtype": "f32", "stats": True},
        # The norm's backward pass in a training step, with both weights' gradients.
        {"name": "norm backward", "op": "norm_backward", "m": 8192, "n": 8192, "dtype": "bf16"},
        # Dropout of a block's output, added to the skip connection.
        {"name": "dropout residual", "op": "dropout", "m": 8192, "n": 4096, "dtype": "bf16", "p": 0.1,
         "residual": True},
        # Its backward pass on an odd fp32 batch: the same mask on the gradient.
        {"name": "dropout backward odd", "op": "dropout_backward", "m": 1237, "n": 1001, "dtype": "f32", "p": 0.25},
    ]


def _size(rng, lo, hi):
    """A length spread over the logarithm of [lo, hi]: round ones, multiples of 8, any."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    step = rng.choice((64, 64, 8, 1))
    return max(lo, min(hi, v // step * step if v >= step else v))


def draw(rng):
    op = rng.choice(("linear", "linear", "linear_backward", "gated", "gated", "gated_backward", "norm", "norm_backward",
                     "dropout", "dropout_backward"))
    if op.startswith(("linear", "gated")):
        while True:
            c = {"op": op, "m": _size(rng, 1, 8192), "k": _size(rng, 64, 8192), "n": _size(rng, 64, 16384),
                 "dtype": rng.choice(("bf16", "bf16", "f16")), "trans_w": rng.random() < 0.5,
                 "act": rng.choice(ACTS if op.startswith("linear") else ACTS[1:])}
            if work(c)["flops"] <= 3.8e12 and (rng.random() < 0.2 or c["m"] * c["k"] * c["n"] > 1 << 24):
                break
        if op in ("linear", "gated"):
            c["bias"] = rng.random() < 0.5
            c["preact"] = c["m"] > 64 and rng.random() < 0.5
        if op == "linear":
            c["residual"] = rng.random() < 0.5
        return c
    dtype = rng.choice(("bf16", "f16", "f32"))
    while True:
        c = {"op": op, "m": _size(rng, 1, 32768), "n": _size(rng, 64, 16384), "dtype": dtype}
        if c["m"] * c["n"] <= 8192 * 8192:
            break
    if op == "norm":
        c["stats"] = rng.random() < 0.5
    elif op.startswith("dropout"):
        c["p"] = rng.choice((0.05, 0.1, 0.2, 0.5))
        if op == "dropout":
            c["residual"] = rng.random() < 0.5
    return c


def work(case):
    m, n, es = case["m"], case["n"], SIZE[case["dtype"]]
    op = case["op"]
    if op.startswith(("linear", "gated")):
        k = case["k"]
        wide = 2 * n if op.startswith("gated") else n  # columns of the weights and of the pre-activation
        if op.endswith("backward"):
            # dy, x, w and the pre-activation in; dx, dw and db out; two products
            z = m * wide if op.startswith("gated") or case["act"] != "none" else 0
            return {"bytes": es * (m * n + 2 * m * k + 2 * k * wide + z + wide), "flops": 4.0 * m * k * wide}
        out = m * n + (m * wide if case.get("preact") else 0)
        inp = m * k + k * wide + (wide if case.get("bias") else 0) + (m * n if case.get("residual") else 0)
        return {"bytes": es * (inp + out), "flops": 2.0 * m * k * wide}
    if op == "norm":
        return {"bytes": es * (2 * m * n + 2 * n) + (8 * m if case["stats"] else 0), "flops": 8.0 * m * n}
    if op == "norm_backward":
        return {"bytes": es * (3 * m * n + 3 * n) + 8 * m, "flops": 14.0 * m * n}
    return {"bytes": es * m * n * (3 if case.get("residual") else 2), "flops": 2.0 * m * n}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    m, n, op = case["m"], case["n"], case["op"]

    def normal(*shape, scale=1.0, to=dt):
        return (torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * scale).to(to)

    s = {"case": case}
    if op.startswith(("linear", "gated")):
        k = case["k"]
        wide = 2 * n if op.startswith("gated") else n
        s["x"] = normal(m, k)
        s["w"] = normal(wide, k, scale=k ** -0.5) if case["trans_w"] else normal(k, wide, scale=k ** -0.5)
        if op.endswith("backward"):
            s["dy"] = normal(m, n, scale=0.25)
            # what the forward pass kept (its bias left out: the gradients do not read it)
            if op.startswith("gated") or case["act"] != "none":
                s["z"] = s["x"] @ (s["w"].t() if case["trans_w"] else s["w"])
        else:
            if case["bias"]:
                s["bias"] = normal(wide, scale=0.3)
            if case.get("residual"):
                s["residual"] = normal(m, n)
        return s
    if op.startswith("norm"):
        # a few channels are far larger than the others, as in a residual stream
        x = torch.randn(m, n, generator=g, device="cuda") * 0.8 + 0.1
        x[:, :: max(1, n // 4 + 1)] *= 12.0
        s["x"] = x.to(dt)
        s["weight"] = (1 + normal(n, scale=0.2, to=torch.float32)).to(dt)
        if op == "norm":
            s["bias"] = normal(n, scale=0.2)
        else:
            s["dy"] = normal(m, n, scale=0.25)
            xd = s["x"].double()
            s["mean"] = xd.mean(1).float()
            s["rstd"] = (xd.var(1, unbiased=False) + 1e-5).rsqrt().float()
        return s
    s["x"] = normal(m, n)
    s["seed"] = int(seed) * 2654435761 % (1 << 40) + 17
    s["offset"] = int(seed) % 1000 * 4097
    if case.get("residual"):
        s["residual"] = normal(m, n)
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


def _act_grad(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    if act == "sigmoid":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 - s)
    return torch.ones_like(z)


def _keep(count, seed, offset, p, device):
    """Philox4x32-10 (Salmon et al., 2011): key `seed`, counter offset + i // 4, word i % 4 of
    the result for element i; an element is kept when its word is at least round(p * 2^32)."""
    low = 0xFFFFFFFF
    i = torch.arange((count + 3) // 4, device=device, dtype=torch.int64) + offset
    c0, c1 = i & low, (i >> 32) & low
    c2, c3 = torch.zeros_like(i), torch.zeros_like(i)
    k0, k1 = seed & low, (seed >> 32) & low
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # 64-bit products; the bits wrap, none is lost
        c0, c1, c2, c3 = ((p1 >> 32) & low) ^ c1 ^ k0, p1 & low, ((p0 >> 32) & low) ^ c3 ^ k1, p0 & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack((c0, c1, c2, c3), 1).reshape(-1)[:count] >= int(round(p * 2.0 ** 32))


def _plain(s):
    c = s["case"]
    op, dt = c["op"], DTYPES[c["dtype"]]
    n = c["n"]
    if op.startswith(("linear", "gated")):
        x, w = s["x"].float(), s["w"].float()
        if c["trans_w"]:
            w = w.t()
        if op.endswith("backward"):
            dy = s["dy"].float()
            if op == "linear_backward":
                dz = dy * _act_grad(s["z"].float(), c["act"]) if "z" in s else dy
            else:
                a, b = s["z"][:, :n].float(), s["z"][:, n:].float()
                dz = torch.cat((dy * b * _act_grad(a, c["act"]), dy * _act(a, c["act"])), 1)
            dw = dz.t() @ x if c["trans_w"] else x.t() @ dz
            return [(dz @ w.t()).to(dt), dw.to(dt), dz.sum(0).to(dt)]
        z = x @ w
        if "bias" in s:
            z = z + s["bias"].float()
        y = _act(z, c["act"]) if op == "linear" else _act(z[:, :n], c["act"]) * z[:, n:]
        if "residual" in s:
            y = y + s["residual"].float()
        return [y.to(dt), z.to(dt)] if c["preact"] else [y.to(dt)]
    if op == "norm":
        x = s["x"].float()
        mean = x.mean(1, keepdim=True)
        d = x - mean
        rstd = 1 / torch.sqrt((d * d).mean(1, keepdim=True) + 1e-5)
        y = (d * rstd * s["weight"].float() + s["bias"].float()).to(dt)
        return [y, mean[:, 0], rstd[:, 0]] if c["stats"] else [y]
    if op == "norm_backward":
        rstd = s["rstd"][:, None]
        h = (s["x"].float() - s["mean"][:, None]) * rstd
        dy = s["dy"].float()
        t = dy * s["weight"].float()
        dx = rstd * (t - t.mean(1, keepdim=True) - h * (t * h).mean(1, keepdim=True))
        return [dx.to(dt), (dy * h).sum(0).to(dt), dy.sum(0).to(dt)]
    x = s["x"].float()
    keep = _keep(x.numel(), s["seed"], s["offset"], c["p"], x.device).view(x.shape)
    y = torch.where(keep, x * (1 / (1 - c["p"])), torch.zeros_like(x))
    if "residual" in s:
        y = y + s["residual"].float()
    return [y.to(dt)]


# ------------------------------------------------------------------ the framework's calls
def _own(s):
    import cuop_b200 as cx

    c = s["case"]
    op = c["op"]
    if op == "linear":
        if c["preact"]:
            z = s["x"].new_empty((c["m"], c["n"]))
            return [cx.linear(s["x"], s["w"], s.get("bias"), s.get("residual"), activation=c["act"],
                              trans_w=c["trans_w"], preact=z), z]
        return [cx.linear(s["x"], s["w"], s.get("bias"), s.get("residual"), activation=c["act"],
                          trans_w=c["trans_w"])]
    if op == "linear_backward":
        return list(cx.linear_backward(s["dy"], s["x"], s["w"], s.get("z"), activation=c["act"],
                                       trans_w=c["trans_w"]))
    if op == "gated":
        if c["preact"]:
            z = s["x"].new_empty((c["m"], 2 * c["n"]))
            return [cx.gated_linear(s["x"], s["w"], s.get("bias"), activation=c["act"], trans_w=c["trans_w"],
                                    preact=z), z]
        return [cx.gated_linear(s["x"], s["w"], s.get("bias"), activation=c["act"], trans_w=c["trans_w"])]
    if op == "gated_backward":
        return list(cx.gated_linear_backward(s["dy"], s["x"], s["w"], s["z"], activation=c["act"],
                                             trans_w=c["trans_w"]))
    if op == "norm":
        if c["stats"]:
            mean, rstd = (torch.empty(c["m"], device="cuda") for _ in range(2))
            return [cx.layer_norm(s["x"], s["weight"], s["bias"], eps=1e-5, mean=mean, rstd=rstd), mean, rstd]
        return [cx.layer_norm(s["x"], s["weight"], s["bias"], eps=1e-5)]
    if op == "norm_backward":
        return list(cx.layer_norm_backward(s["dy"], s["x"], s["mean"], s["rstd"], s["weight"]))
    if op == "dropout":
        return [cx.dropout(s["x"], c["p"], s["seed"], s["offset"], residual=s.get("residual"))]
    return [cx.dropout_backward(s["x"], c["p"], s["seed"], s["offset"])]


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------ the definitions in 64 bits
def _phi(z):
    """The normal distribution function."""
    return 0.5 * torch.special.erfc(-z / math.sqrt(2.0))


def _sig(z):
    return 0.5 * (torch.tanh(0.5 * z) + 1)


def _value_and_slope(z, act):
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        return z.clamp_min(0), torch.heaviside(z, torch.zeros_like(z))
    if act == "sigmoid":
        return _sig(z), _sig(z) * _sig(-z)
    if act == "silu":
        return z * _sig(z), _sig(z) + z * _sig(z) * _sig(-z)
    if act == "gelu":
        return z * _phi(z), _phi(z) + z * torch.exp(-z.square() / 2) / math.sqrt(2 * math.pi)
    # gelu_tanh: 0.5 (1 + tanh u) = sigmoid(2u)
    u2 = 2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)
    du2 = 2 * math.sqrt(2 / math.pi) * (1 + 0.134145 * z ** 2)
    return z * _sig(u2), _sig(u2) + z * _sig(u2) * _sig(-u2) * du2


def _words(count, seed, offset):
    """The generator's words with 16-bit limbs: no product exceeds 2^49."""
    def mul(a, b):
        bl, bh = b & 0xFFFF, b >> 16
        lo, hi = a * bl, a * bh
        t = lo + ((hi & 0xFFFF) << 16)
        return (t >> 32) + (hi >> 16), t % (1 << 32)

    ctr = torch.arange(offset, offset + -(-count // 4), dtype=torch.int64, device="cuda")
    v = [ctr % (1 << 32), ctr // (1 << 32), 0 * ctr, 0 * ctr]
    for r in range(10):
        ka, kb = (seed + r * 0x9E3779B9) % (1 << 32), ((seed >> 32) + r * 0xBB67AE85) % (1 << 32)
        ah, al = mul(v[0], 0xD2511F53)
        bh, bl = mul(v[2], 0xCD9E8D57)
        v = [bh ^ v[1] ^ ka, bl, ah ^ v[3] ^ kb, al]
    return torch.cat([t[:, None] for t in v], dim=1).flatten()[:count]


def exact(case, seed):
    s = prepare(case, seed)
    op, n = case["op"], case["n"]
    d = {k: v.double() for k, v in s.items() if isinstance(v, torch.Tensor)}
    if op.startswith(("linear", "gated")):
        w = d["w"].mT if case["trans_w"] else d["w"]
        if op.endswith("backward"):
            if op == "linear_backward":
                dz = d["dy"] * (_value_and_slope(d["z"], case["act"])[1] if "z" in d else 1)
            else:
                v, slope = _value_and_slope(d["z"][:, :n], case["act"])
                dz = torch.hstack((d["dy"] * d["z"][:, n:] * slope, d["dy"] * v))
            dw = torch.mm(d["x"].mT, dz)
            return [torch.mm(dz, w.mT), dw.mT.contiguous() if case["trans_w"] else dw, dz.sum(0)]
        z = torch.mm(d["x"], w) + d.get("bias", 0)
        if op == "linear":
            y = _value_and_slope(z, case["act"])[0]
        else:
            y = _value_and_slope(z[:, :n], case["act"])[0] * z[:, n:]
        y = y + d.get("residual", 0)
        return [y, z] if case["preact"] else [y]
    if op == "norm":
        var, mean = torch.var_mean(d["x"], 1, correction=0)
        y = torch.addcmul(d["bias"], (d["x"] - mean[:, None]) / torch.sqrt(var + 1e-5)[:, None], d["weight"])
        return [y, mean, (var + 1e-5) ** -0.5] if case["stats"] else [y]
    if op == "norm_backward":
        h = (d["x"] - d["mean"][:, None]) * d["rstd"][:, None]
        t = d["dy"] * d["weight"]
        # the projections of t on the constant row and on h leave it
        dx = t - t.sum(1, keepdim=True) / n - h * ((t * h).sum(1, keepdim=True) / n)
        return [dx * d["rstd"][:, None], torch.einsum("ij,ij->j", d["dy"], h), d["dy"].sum(0)]
    drop = _words(d["x"].numel(), s["seed"], s["offset"]).view(d["x"].shape) < int(round(case["p"] * 4294967296.0))
    y = (d["x"] / (1 - case["p"])).masked_fill(drop, 0.0)
    return [y + d.get("residual", 0)]
