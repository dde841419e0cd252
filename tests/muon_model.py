"""The Muon program's arithmetic restated on the host: what its f16 parts and its tensor-core sums may cost, for tolerances that see a
missing low half."""
import numpy as np

from tests import operators_ref as R

SCALE = 1024.0          # operands are multiplied by it, so that their parts stay inside f16's normal range
CHUNK, SLICE = 128, 16  # of the contraction: summed in one accumulator, per instruction


def parts(x, n):
    """x as n f16 numbers whose sum is nearly x"""
    out, rest = [], np.asarray(x, np.float64) * SCALE
    for _ in range(n):
        p = rest.astype(np.float32).astype(np.float16).astype(np.float64)
        out.append(p / SCALE)
        rest = rest - p
    return out


def truncated(x):
    """x with 24 bits, towards zero: how an accumulator takes a sum"""
    m, e = np.frexp(x)
    return np.ldexp(np.trunc(m * 2.0 ** 24), e - 24)


def product(a, b, dropped=()):
    """The sum of a_i b_j over the parts without the product of the two low halves, added as the kernels add: per chunk of the
    contraction in one accumulator, slice by slice and the small products first, the chunks in f32.  dropped: pairs (i, j) left out."""
    if len(a) == 1:
        return a[0] @ b[0]
    pairs = [p for p in ((1, 0), (0, 1), (0, 0)) if p not in dropped]
    k = a[0].shape[1]
    total = np.zeros((a[0].shape[0], b[0].shape[1]), np.float32)
    for c in range(0, k, CHUNK):
        acc = np.zeros(total.shape)
        for s in range(c, min(k, c + CHUNK), SLICE):
            e = min(k, s + SLICE)
            for i, j in pairs:
                acc = truncated(acc + a[i][:, s:e] @ b[j][s:e])
        total += acc.astype(np.float32)
    return total.astype(np.float64)


def direction(u, n, steps=5, abc=R.NS, eps=1e-7, dropped=((), (), ())):
    """The step made from u with every operand held as n parts.  dropped: per product (gram, polynomial, result) the pairs left out."""
    a, b, c = abc
    tall = u.shape[0] > u.shape[1]
    x = u.T if tall else u
    x = parts(x / (np.linalg.norm(x) + eps), n)
    for _ in range(steps):
        gram = parts(product(x, [p.T for p in x], dropped[0]), n)
        poly = parts(a * np.eye(len(gram[0])) + b * sum(gram) + c * product(gram, gram, dropped[1]), n)
        x = parts(product(poly, x, dropped[2]), n)
    x = sum(x)
    return x.T if tall else x


def exact(u, steps=5, abc=R.NS, eps=1e-7):
    a, b, c = abc
    tall = u.shape[0] > u.shape[1]
    x = u.T if tall else u
    x = x / (np.linalg.norm(x) + eps)
    for _ in range(steps):
        gram = x @ x.T
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.T if tall else x


def single_part_error(u, want, **kw):
    """Of operands held as one f16 each, in the Frobenius norm.  The 16-bit programs make it once (their sums are f32: the truncation of
    at most 256 additions is 2^-16 of a sum, below f16's 2^-11), f32 programs have to stay a factor of 16 below."""
    return float(np.linalg.norm(direction(u, 1, **kw) - want))


ONE_PART, TWO_PARTS = 2.0, 1.0 / 16
