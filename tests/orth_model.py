"""The Newton-Schulz iteration in 64 bits, in fp32, and on operands cut to fp16 halves, all with the default coefficients
unless given: what the orthogonalisation's errors are compared with."""
import torch

COEFFS = (3.4445, -4.7750, 2.0315)


def iterate(G, steps, coeffs=COEFFS, eps=1e-7, dtype=torch.float64):
    """The iteration with torch's products of `dtype`, the input scaled in 64 bits."""
    a, b, c = coeffs
    X = G.double()
    X = (X / (X.norm() + eps)).to(dtype)
    flip = X.shape[0] > X.shape[1]
    X = X.t().contiguous() if flip else X
    for _ in range(steps):
        A = X @ X.t().contiguous()
        X = a * X + (b * A + c * (A @ A)) @ X
    return X.t() if flip else X


def halves(x, e):
    v = (x.float() * 2.0 ** e).float()
    hi = v.half()
    lo = (v - hi.float()).half()
    return hi.double() / 2.0 ** e, lo.double() / 2.0 ** e


def split_iterate(G, steps, terms, coeffs=COEFFS, eps=1e-7):
    """Operands in two fp16 halves (2^12 X and A, 2^11 B), their products the sum of `terms` pairs of halves."""
    a, b, c = coeffs
    product = lambda p, q: sum(p[i] @ q[j].t().contiguous() for i, j in terms).float()  # noqa: E731
    X = G.double()
    X = (X / (X.norm() + eps)).float()
    flip = X.shape[0] > X.shape[1]
    X = X.t().contiguous() if flip else X
    for _ in range(steps):
        x = halves(X, 12)
        A = halves(product(x, x), 12)
        B = halves((b * (A[0] + A[1]) + c * product(A, A).double()).float(), 11)
        X = (a * (x[0] + x[1]) + product(B, [h.t() for h in x]).double()).float()
    return X.t() if flip else X


def error(out, ref):
    """Relative to the reference, in the Frobenius norm."""
    return float((out.double() - ref).norm() / ref.norm())


def bound(G, ref, steps, **kw):
    """A regression bound, found by measurement and not by a proof: four times what fp32 products leave on the same input
    (kernel and torch differ by the order of their sums only; measured 0.4 to 1.1 times), at least 2^-21."""
    return max(4.0 * error(iterate(G, steps, dtype=torch.float32, **kw), ref), 2.0 ** -21)


def graded(m, n, scale, seed=0):
    """Half of the rows `scale` times the others."""
    G = torch.randn(m, n, generator=torch.Generator().manual_seed(seed))
    G[m // 2:] *= scale
    return G
