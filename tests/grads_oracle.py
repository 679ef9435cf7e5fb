"""Plain restatement of the optimiser's operators over lists of gradients in extended precision (x87 80-bit where numpy has it), and the bounds
that float64 arithmetic may be off by."""
import math
import numpy as np

U = 2.0 ** -53                       # half a step of float64: what one rounding may be off by, relative
LD = np.longdouble


def real_view(a):
    a = np.ascontiguousarray(a).reshape(-1)
    return a.view(np.float64) if a.dtype == np.complex128 else a


def norms(arrays):
    """(2-norm, largest modulus) as longdouble: exponent range and precision beyond float64's, so squares neither overflow nor underflow."""
    s, top = LD(0), LD(0)
    for a in arrays:
        x = real_view(a).astype(LD)
        s += (x * x).sum()
        if a.size:
            m = np.sqrt((x.reshape(-1, 2) ** 2).sum(1)) if a.dtype == np.complex128 else np.abs(x)
            top = max(top, m.max())
    return np.sqrt(s), top


def tol_n2(n):
    """Relative bound on the 2-norm of n doubles.  Every square sum is of non-negative terms, so each addition or fused product costs a relative U
    of the result at most: per thread the pairs of its chunks (n / (2 * 256) over at most 1024 workgroups, and up to 4 more for the short chunk
    at the end of each of the tensors it meets, fewer than 16 here), 2 roundings of a pair's own squares, 6 levels of the wave, up to 16 of the
    workgroup, 5 + 6 + 3 of the last combination; half of it through the root, one rounding of the root, one of the scaling by a power of two."""
    depth = n / (2.0 * 256 * 1024) + 64 + 2 + 6 + 16 + 14
    return (depth / 2 + 2) * U


def tol_top(cplx):
    return 3 * U if cplx else 0.0        # |z|^2: 2 roundings, halved by the root; the root itself; one of the reference's conversion


def factor(n, max_norm):
    return LD(1) if n <= max_norm else LD(max_norm) / n


def f64(x):
    return float(x)
