"""Plain 64-bit forms of the embedding, RMS norm and Muon programs, the storage types, and what one rounding may cost."""
import numpy as np

from zyx_b200 import _lib as L

NP = {L.F32: np.float32, L.BF16: np.uint16, L.F16: np.uint16}
DTYPES = [L.F32, L.BF16, L.F16]
NAMES = {L.F32: "f32", L.BF16: "bf16", L.F16: "f16"}
HALF_STEP = {L.F32: 2.0 ** -24, L.BF16: 2.0 ** -8, L.F16: 2.0 ** -11}     # of the value, rounding to nearest
F32 = 2.0 ** -24
F16_TINY = {True: 2.0 ** -25, False: 2.0 ** -14}      # f16 below its normal range: half a subnormal step; flushed to zero when truncating


def unit(dtype, nearest):
    """Relative error of one store: half a step to nearest, a whole one when 16-bit stores truncate."""
    return HALF_STEP[dtype] * (1 if nearest or dtype == L.F32 else 2)


def tiny(dtype, nearest):
    """Absolute error of one store near zero."""
    return F16_TINY[nearest] if dtype == L.F16 else 2.0 ** -133 if dtype == L.BF16 else 2.0 ** -149


def store(x, dtype):
    """float64 -> storage bits, to nearest even."""
    x32 = np.ascontiguousarray(x, np.float32)
    if dtype == L.F32:
        return x32
    if dtype == L.F16:
        return x32.astype(np.float16).view(np.uint16)
    b = x32.view(np.uint32)
    out = ((b + 0x7fff + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x32), np.uint16(0x7fc0), out)


def value(bits, dtype):
    """storage bits -> float64"""
    if dtype == L.F32:
        return np.asarray(bits, np.float64)
    if dtype == L.F16:
        return np.ascontiguousarray(bits).view(np.float16).astype(np.float64)
    return (np.ascontiguousarray(bits).astype(np.uint32) << 16).view(np.float32).astype(np.float64)


E4M3 = np.zeros(256)
for _b in range(256):
    _e, _m = (_b >> 3) & 15, _b & 7
    _v = (_m / 8.0) * 2.0 ** -6 if _e == 0 else (1 + _m / 8.0) * 2.0 ** (_e - 7)
    E4M3[_b] = np.nan if (_b & 127) == 127 else (-_v if _b & 128 else _v)


def close(got, want, tol):
    """got and want float64, tol the largest permitted difference of each element; NaN has to meet NaN, infinities the same."""
    got, want, tol = np.broadcast_arrays(np.asarray(got, np.float64), np.asarray(want, np.float64), np.asarray(tol, np.float64))
    odd = ~np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), "NaN in other places"
    keep = odd & ~np.isnan(want)
    assert np.array_equal(got[keep], want[keep]), "infinities differ"
    diff = np.abs(got[~odd] - want[~odd])
    bad = diff > tol[~odd]
    if bad.any():
        i = int(np.argmax(diff - tol[~odd]))
        raise AssertionError("%d of %d out of tolerance; worst: got %r, want %r, tolerance %r" %
                             (int(bad.sum()), diff.size, got[~odd][i], want[~odd][i], tol[~odd][i]))


# ---- embedding ----
def embedding(ids, table, scale=1.0):
    out = np.zeros((ids.size, table.shape[1]))
    met = (ids >= 0) & (ids < table.shape[0])
    out[met] = table[ids[met]] * scale
    return out


def embedding_bwd(ids, dout, vocab, scale=1.0):
    """-> the gradient and, for its tolerance, the sum of magnitudes and the number of terms of each row"""
    total, mags, terms = np.zeros((vocab, dout.shape[1])), np.zeros((vocab, dout.shape[1])), np.zeros((vocab, 1))
    met = np.nonzero((ids >= 0) & (ids < vocab))[0]
    np.add.at(total, ids[met], dout[met] * scale)
    np.add.at(mags, ids[met], np.abs(dout[met] * scale))
    np.add.at(terms, ids[met], 1)
    return total, mags, terms


# ---- RMS norm ----
def rmsnorm(x, residual, weight, eps):
    h = x + residual if residual is not None else x
    with np.errstate(all="ignore"):
        y = h / np.sqrt(np.mean(h * h, axis=1, keepdims=True) + eps)
        return h, y * weight if weight is not None else y


def rmsnorm_bwd(h, dy, weight, dh, eps):
    """-> dx, dweight and the magnitudes their errors scale with"""
    n = h.shape[1]
    with np.errstate(all="ignore"):
        rstd = 1.0 / np.sqrt(np.mean(h * h, axis=1, keepdims=True) + eps)
        g = dy * weight if weight is not None else dy
        xh = h * rstd
        dx = rstd * (g - xh * np.mean(g * xh, axis=1, keepdims=True))
        size = rstd * (np.abs(g) + np.abs(xh) * np.sum(np.abs(g * xh), axis=1, keepdims=True) / n)
        if dh is not None:
            dx, size = dx + dh, size + np.abs(dh)
        return dx, (dy * xh).sum(0), size, np.abs(dy * xh).sum(0)


# ---- Muon ----
NS = (3.4445, -4.7750, 2.0315)


def slope(sigma, abc):
    """Largest factor by which X -> aX + (bA + cA^2)X stretches a small change of X with these singular values: the divided
    differences of the odd polynomial, (p(s) - p(t)) / (s - t) and (p(s) + p(t)) / (s + t)."""
    a, b, c = abc
    s = np.unique(np.concatenate([sigma, [0.0]]))
    if s.size > 300:
        s = s[np.linspace(0, s.size - 1, 300).astype(int)]
    s, t = s[:, None], s[None, :]
    minus = a + b * (s * s + s * t + t * t) + c * (s ** 4 + s ** 3 * t + s * s * t * t + s * t ** 3 + t ** 4)
    plus = a + b * (s * s - s * t + t * t) + c * (s ** 4 - s ** 3 * t + s * s * t * t - s * t ** 3 + t ** 4)
    return float(max(np.abs(minus).max(), np.abs(plus).max()))


def orthogonalise(u, steps=5, abc=NS, eps=1e-7, rounding=0.0):
    """-> X after the steps, and a bound of the Frobenius norm of its error when X, A and the polynomial of A are each rounded with
    relative error `rounding` in every step."""
    a, b, c = abc
    tall = u.shape[0] > u.shape[1]
    x = u.T if tall else u
    x = x / (np.linalg.norm(x) + eps)
    err = rounding * np.linalg.norm(x)
    for _ in range(steps):
        sigma = np.linalg.svd(x, compute_uv=False)
        top = sigma[0] if sigma.size else 0.0
        gram = x @ x.T
        poly = a * np.eye(x.shape[0]) + b * gram + c * gram @ gram
        nxt = poly @ x
        # A: rounded once; bA + cA^2: the change of A goes through it, then it is rounded; the product is rounded again
        d_gram = rounding * np.linalg.norm(gram)
        d_poly = (abs(b) + 2 * abs(c) * top * top) * d_gram + rounding * np.linalg.norm(poly)
        err = slope(sigma, abc) * err + d_poly * top + rounding * np.linalg.norm(nxt)
        x = nxt
    return (x.T if tall else x), err


def adjust(kind, rows, cols):
    return 0.2 * np.sqrt(max(rows, cols)) if kind == L.MUON_ADJUST_RMS else np.sqrt(max(1.0, rows / cols))
