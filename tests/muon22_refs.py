"""How far the Newton-Schulz kernels may be off where the products' operands keep 22 bits.

What rounds then, a step (the state X, A = X X^T, the polynomial P; muon_refs.py maps an error of each to the result):
  - a product's sums, held in fp32 by tensor cores whose rounding nothing specifies but that no addition loses more
    than 2^-23 of the running sum: n = depth / 16 + 4 additions (sixteen terms enter at a time), which may all fall the
    same way, so n 2^-23 of the running sums' size.  A sum that starts at nothing, ends at S and is made of increments
    d_k runs at no more than about S and a random walk of the increments: R^2 = ||S||^2 + sum ||d_k||^2;
  - the terms lo lo that are left out: each lo is 2^-11 of its hi at most, 2^-11 / sqrt(12) on average: 2^-22 / 12 R;
  - X, A and P as hi + lo: 2^-22 of an element at most, each; and three fp32 operations on the way, 2^-24 each.
"""
import torch

import muon_refs as R


def _walk(a, b):
    """(sum over k of ||a_k||^2 ||b_k||^2) of a product's increments, a's columns times b's rows."""
    return float(((a * a).sum(0) * (b * b).sum(1)).sum())


def predicted22(x, coefficients, singular=None):
    """Bound (Frobenius norm) of the error of the iteration from x, one matrix in 64 bits, errors of products spread evenly."""
    s = torch.linalg.svdvals(x) if singular is None else singular
    if x.shape[0] > x.shape[1]:
        x = x.mT
    p, q = x.shape
    v = torch.zeros(p, p, dtype=torch.float64, device=x.device)
    vx = torch.zeros(p, dtype=torch.float64, device=x.device)
    own = (2.0 ** -22 + 3 * 2.0 ** -24) ** 2

    def sums(norm2, walk, depth):
        r2 = norm2 + walk
        return ((depth / 16 + 4) * 2.0 ** -23 + 2.0 ** -22 / 12) ** 2 * r2

    for a, b, c in coefficients:
        t = s * s
        f, g = (lambda z: a * z + b * z ** 3 + c * z ** 5), (lambda z: b * z ** 3 + c * z ** 5)
        one, other = R._quotients(f, s)
        v = one ** 2 * v + other ** 2 * v.t()
        ratio = a + b * t + c * t * t
        vx = ratio ** 2 * vx
        # X as the products read it
        x_var = own * float(t.sum()) / (p * q)
        one, other = R._quotients(g, s)
        v = v + (one ** 2 + other ** 2) * x_var
        vx = vx + (ratio - a) ** 2 * x_var
        gram = x @ x.mT
        poly = b * gram + c * (gram @ gram)
        a_norm2, p_norm2 = float((t * t).sum()), float(((b * t + c * t * t) ** 2).sum())
        a_var = (own * a_norm2 + sums(a_norm2, _walk(x, x.mT), q)) / (p * p)
        v = v + a_var * ((b + c * (t[:, None] + t[None, :])) * s[None, :]) ** 2
        p_var = (own * p_norm2 + c * c * sums(float((t ** 4).sum()), _walk(gram, gram), p)) / (p * p)
        v = v + p_var * s[None, :] ** 2
        done = a * x + poly @ x
        u_var = (own * float((done * done).sum()) + sums(float(((poly @ x) ** 2).sum()), _walk(poly, x), p)) / (p * q)
        v, vx = v + u_var, vx + u_var
        x, s = done, f(s).abs()
    return float((v.sum() + (q - p) * vx.sum()).sqrt())


def allowed22(x, coefficients, dtype, singular=None):
    """Three times that from 16 rows on, ten times below, where errors are not spread; and the result's own rounding."""
    p = min(x.shape)
    return (3.0 if p >= 16 else 10.0) * predicted22(x, coefficients, singular) + \
        (torch.finfo(dtype).eps / 2 + 3 * 2.0 ** -23) * float(torch.linalg.matrix_norm(R.iterate(x, coefficients)))
