"""Newton-Schulz iteration and Muon step in 64 bits, and how far the kernels may be off.

The kernels round to fp16 at three places a step (u = 2^-11): the operand X of
the products (aX itself keeps 22 bits), A = X X^T, and the polynomial P.  A
rounding of v is uniform over half a spacing either way, so its variance is
spacing^2 / 12: 0.18 u^2 v^2 on average over a binade.  In the basis of X's
singular vectors a step maps an error's entry (i, j), i and j both below p, by
the divided differences of f(s) = a s + b s^3 + c s^5,
  (f_i - f_j) / (s_i - s_j)  on its symmetric,
  (f_i + f_j) / (s_i + s_j)  on its antisymmetric part,
and the entries beyond by f_i / s_i.  predicted() follows the variances through
the steps.  The sums' own errors, 2^-23 each, are far below.
"""
import torch

COEFFICIENTS = (3.4445, -4.7750, 2.0315)
U = 2.0 ** -11
VAR = 0.18 * U * U


def normalised(g, eps=1e-7):
    g = g.double()
    return g / (torch.linalg.matrix_norm(g, keepdim=True) + eps)


def step(x, k):
    a, b, c = k
    if x.shape[-2] > x.shape[-1]:
        t = x.mT @ x
        return a * x + x @ (b * t + c * (t @ t))
    t = x @ x.mT
    return a * x + (b * t + c * (t @ t)) @ x


def iterate(x, coefficients):
    for k in coefficients:
        x = step(x, k)
    return x


def _quotients(f, s):
    """Factors of an entry by itself and by its mirror image, for f(s) given at s."""
    d = s[:, None] - s[None, :]
    same = d.abs() < 1e-9 * (s[:, None] + s[None, :] + 1e-300)
    minus = (f(s)[:, None] - f(s)[None, :]) / torch.where(same, torch.ones_like(d), d)
    h = 1e-6 * (s + 1e-12)
    slope = (f(s + h) - f(s - h)) / (2 * h)
    minus = torch.where(same, slope[:, None].expand_as(d), minus)
    total = (s[:, None] + s[None, :]).clamp_min(1e-300)
    plus = (f(s)[:, None] + f(s)[None, :]) / total
    return (minus + plus) / 2, (minus - plus) / 2


def predicted(x, coefficients):
    """Root mean square (Frobenius norm) of the error of the iteration from x, one matrix in 64 bits."""
    s = torch.linalg.svdvals(x)
    p, q = min(x.shape), max(x.shape)
    v = torch.zeros(p, p, dtype=torch.float64, device=x.device)
    vx = torch.zeros(p, dtype=torch.float64, device=x.device)  # of each entry beyond column p
    for a, b, c in coefficients:
        t = s * s
        f, g = (lambda z: a * z + b * z ** 3 + c * z ** 5), (lambda z: b * z ** 3 + c * z ** 5)
        one, other = _quotients(f, s)
        v = one ** 2 * v + other ** 2 * v.t()
        ratio = a + b * t + c * t * t
        vx = ratio ** 2 * vx
        x_var = VAR * float((s * s).sum()) / (p * q)
        one, other = _quotients(g, s)
        v = v + (one ** 2 + other ** 2) * x_var
        vx = vx + (ratio - a) ** 2 * x_var
        poly = b * t + c * t * t
        a_var = VAR * float((t * t).sum()) / (p * p)
        v = v + a_var * ((b + c * (t[:, None] + t[None, :])) * s[None, :]) ** 2
        v = v + VAR * float((poly * poly).sum()) / (p * p) * s[None, :] ** 2
        s = f(s).abs()
    return float((v.sum() + (q - p) * vx.sum()).sqrt())


def allowed(x, coefficients, dtype):
    """Largest Frobenius norm of the error that counts as right: three times the
    predicted one, ten times below 16 rows, where a few roundings, each up to 2.4 times
    its root mean square, do not average; plus the result's own rounding, the
    22 bits of X (2^-22) and the fp32 factors that scale it in and out (2^-23)."""
    p = min(x.shape)
    return (3.0 if p >= 16 else 10.0) * predicted(x, coefficients) + \
        (torch.finfo(dtype).eps / 2 + 3 * 2.0 ** -23) * float(torch.linalg.matrix_norm(iterate(x, coefficients)))


def allowed_equal(s, coefficients):
    """The same for a matrix of equal elements, whose one singular value is s: all elements of a matrix round the same way,
    so nothing averages.  Each rounding is u at most and moves the one singular value: X's in the products by g'(s) s u,
    A's by (b + 2 c t) t s u, P's by (b t + c t^2) s u; later steps multiply by f'(s).  1 % for products of errors."""
    e = 0.0
    for a, b, c in coefficients:
        t = s * s
        g1 = 3 * b * t + 5 * c * t * t
        e = abs(a + g1) * e + U * s * (abs(g1) + abs(b + 2 * c * t) * t + abs(b * t + c * t * t))
        s = abs(a * s + b * s ** 3 + c * s ** 5)
    return 1.01 * e + 4 * 2.0 ** -23 * s


def rounded_iteration(x, coefficients):
    """The iteration with the kernels' roundings to fp16 put in (scales aside), for the tests of predicted()."""
    def half(v):
        top = v.abs().max().clamp_min(1e-300)
        k = torch.exp2(14 - torch.ceil(torch.log2(top)))
        return (v * k).to(torch.float16).double() / k

    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    for a, b, c in coefficients:
        h = half(x)
        t = half(h @ h.mT)
        x = a * x + half(b * t + c * (t @ t)) @ h
    return x.mT if tall else x
