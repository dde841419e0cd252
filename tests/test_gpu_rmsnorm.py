"""RMS norm (residual, weight, 8-bit output) and its adjoint against 64-bit forms.

Tolerances, in half steps of f32 (2^-24): h is off by 1, a sum of squares by its depth - at most 32 terms in a thread, 10 levels
across a row's threads, 4 for the product, the mean and eps - so y by half of 46 + 3 for the root and the quotient + 3 for the
products + 1 for h: below 40.  In the adjoint the same holds for each factor: rstd, twice rstd and the row product (46 of the sum
of magnitudes), a few products: below 120 of the sum of the terms' magnitudes.  Each store costs one rounding.
"""
import numpy as np
import pytest

from tests import operators_ref as R
from zyx_b200 import _lib as L
from zyx_b200 import backend as B

pytestmark = pytest.mark.gpu
Y_STEPS, DX_STEPS = 40, 120


@pytest.fixture(scope="module", params=[True, False], ids=["nearest", "truncate"])
def gsess(request):
    from zyx_b200 import build
    from zyx_b200.ops import Session
    build.build()
    s = Session(device_ids=[0], debug=2, round_nearest=request.param)
    s.nearest = request.param
    yield s
    s.close()


def data(rng, shape, dtype, scale=1.0, mean=0.0):
    return R.store(rng.standard_normal(shape) * scale + mean, dtype)


SHAPES = [(1, 1), (1, 8), (3, 7), (4, 4096), (9, 64), (33, 100), (5, 513), (300, 777), (65, 2048), (3, 5003), (2, 8192), (3, 16384), (2, 16383), (1200, 24)]


@pytest.mark.parametrize("dtype", R.DTYPES, ids=R.NAMES.get)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_forward(gsess, dtype, rows, cols):
    rng = np.random.default_rng(rows * 7 + cols)
    x, r, w = data(rng, (rows, cols), dtype), data(rng, (rows, cols), dtype, 2.0), data(rng, (cols,), dtype, 0.2, 1.0)
    u, t = R.unit(dtype, gsess.nearest), R.tiny(dtype, gsess.nearest)
    for residual, weight in ((r, w), (None, w), (r, None), (None, None)):
        h64, y64 = R.rmsnorm(R.value(x, dtype), None if residual is None else R.value(r, dtype), None if weight is None else R.value(w, dtype), 1e-6)
        got = gsess.rmsnorm(dtype, x, residual, weight)
        if residual is not None:
            h, got = got
            R.close(R.value(h, dtype), h64, np.abs(h64) * (R.F32 + u) * 1.01 + t)
        R.close(R.value(got, dtype), y64, np.abs(y64) * (Y_STEPS * R.F32 + u) * 1.01 + t)


@pytest.mark.parametrize("dtype", R.DTYPES, ids=R.NAMES.get)
@pytest.mark.parametrize("group", [0, 16, 50, 64, 128])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (4, 4096), (9, 64), (33, 100), (300, 777), (5, 5003), (2, 16384), (2, 16383)])
def test_forward_in_8_bits(gsess, dtype, group, rows, cols):
    rng = np.random.default_rng(rows * 5 + cols + group)
    x, r, w = data(rng, (rows, cols), dtype), data(rng, (rows, cols), dtype, 2.0), data(rng, (cols,), dtype, 0.2, 1.0)
    x[0] = 0                                                  # one row of zeros
    r[0] = 0
    h64, y64 = R.rmsnorm(R.value(x, dtype), R.value(r, dtype), R.value(w, dtype), 1e-6)
    h, (q, scales) = gsess.rmsnorm(dtype, x, r, w, quant=True, group=group)
    R.close(R.value(h, dtype), h64, np.abs(h64) * (R.F32 + R.unit(dtype, gsess.nearest)) * 1.01 + R.tiny(dtype, gsess.nearest))
    width = min(group or cols, cols)
    assert scales.shape == (rows, -(-cols // (group or cols)))
    for g in range(scales.shape[1]):
        part = y64[:, g * width:(g + 1) * width]
        want = np.maximum(np.abs(part).max(1), 1e-30) / 448.0
        R.close(scales[:, g], want, want * (Y_STEPS + 2) * R.F32)
        s = scales[:, g:g + 1].astype(np.float64)
        got = R.E4M3[q[:, g * width:(g + 1) * width]] * s
        # half a step of 3 bits behind the leading one, or of the subnormal range
        R.close(got, part, np.maximum(np.abs(part) * 2.0 ** -4, s * 2.0 ** -10) * (1 + 2 ** -10) + np.abs(part) * Y_STEPS * R.F32)
    assert not q[0].any()


@pytest.mark.parametrize("dtype", R.DTYPES, ids=R.NAMES.get)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_backward(gsess, dtype, rows, cols):
    rng = np.random.default_rng(rows * 11 + cols)
    h, dy, w, dh = data(rng, (rows, cols), dtype, 2.0), data(rng, (rows, cols), dtype), data(rng, (cols,), dtype, 0.2, 1.0), data(rng, (rows, cols), dtype)
    u, t = R.unit(dtype, gsess.nearest), R.tiny(dtype, gsess.nearest)
    for weight, add in ((w, dh), (w, None), (None, dh), (None, None)):
        args = [R.value(h, dtype), R.value(dy, dtype), None if weight is None else R.value(w, dtype), None if add is None else R.value(dh, dtype)]
        dx64, dw64, size, dw_size = R.rmsnorm_bwd(*args, 1e-6)
        got = gsess.rmsnorm_bwd(dtype, h, dy, weight, add)
        if weight is not None:
            got, dw = got
            R.close(R.value(dw, dtype), dw64, dw_size * (rows + Y_STEPS) * R.F32 + np.abs(dw64) * u * 1.01 + t)
            assert np.array_equal(dw, gsess.rmsnorm_bwd(dtype, h, dy, weight, add)[1])        # a fixed order
        R.close(R.value(got, dtype), dx64, size * DX_STEPS * R.F32 + np.abs(dx64) * u * 1.01 + t)


def test_backward_against_differences(gsess):
    """Central differences in 64 bits of sum(dy * norm(h)) along a direction, against <dx, d> and <dweight, dw>.
    The kernel's gradients are off by 2^-24 * (120 of the terms' magnitudes); the difference, with a step of 1e-5, by the third
    derivative's share (1e-10 of the curvature) and 2^-53 / 1e-5: both far below."""
    rng = np.random.default_rng(3)
    rows, cols, eps = 6, 65, 1e-5
    h, dy, w, d = (rng.standard_normal(s).astype(np.float32) for s in ((rows, cols), (rows, cols), (cols,), (rows, cols)))
    dw = rng.standard_normal(cols)
    dx, dweight = gsess.rmsnorm_bwd(L.F32, h, dy, w, eps=eps)
    f = lambda hh, ww: float((dy.astype(np.float64) * R.rmsnorm(hh, None, ww, eps)[1]).sum())       # noqa: E731
    h64, w64 = h.astype(np.float64), w.astype(np.float64)
    t = 1e-5
    by_h, by_w = (f(h64 + t * d, w64) - f(h64 - t * d, w64)) / (2 * t), (f(h64, w64 + t * dw) - f(h64, w64 - t * dw)) / (2 * t)
    _, _, size, dw_size = R.rmsnorm_bwd(h64, dy.astype(np.float64), w64, None, eps)
    assert abs(by_h - float((dx * d.astype(np.float64)).sum())) <= float((size * np.abs(d)).sum()) * 2 ** -16
    assert abs(by_w - float((dweight * dw).sum())) <= float((dw_size * np.abs(dw)).sum()) * 2 ** -16


@pytest.mark.parametrize("dtype", R.DTYPES, ids=R.NAMES.get)
@pytest.mark.parametrize("ld", [72, 83])
def test_row_pitch(gsess, dtype, ld):
    """Rows inside wider ones: what lies between them is not written, and not read (NaN there)."""
    rng = np.random.default_rng(ld)
    rows, cols = 41, 64
    x, r, w = data(rng, (rows, ld), dtype), data(rng, (rows, ld), dtype, 2.0), data(rng, (cols,), dtype, 0.2, 1.0)
    nan = R.store(np.array([np.nan]), dtype)[0]
    x[:, cols:] = nan
    r[:, cols:] = nan
    d = B.rmsnorm_desc(dtype, rows, cols, has_weight=True, ld=ld)
    keep = data(rng, (rows, ld), dtype)
    y = gsess.run(d, [x, w], [((rows, ld), R.NP[dtype])], out_init=keep)[0]
    assert np.array_equal(y[:, cols:], keep[:, cols:])
    _, y64 = R.rmsnorm(R.value(x, dtype)[:, :cols], None, R.value(w, dtype), 1e-6)
    u, t = R.unit(dtype, gsess.nearest), R.tiny(dtype, gsess.nearest)
    R.close(R.value(y, dtype)[:, :cols], y64, np.abs(y64) * (Y_STEPS * R.F32 + u) * 1.01 + t)
    d = B.rmsnorm_desc(dtype, rows, cols, ld=ld, backward=True)
    dx = gsess.run(d, [x, r], [((rows, ld), R.NP[dtype])], out_init=keep)[0]
    assert np.array_equal(dx[:, cols:], keep[:, cols:])
    dx64, _, size, _ = R.rmsnorm_bwd(R.value(x, dtype)[:, :cols], R.value(r, dtype)[:, :cols], None, None, 1e-6)
    R.close(R.value(dx, dtype)[:, :cols], dx64, size * DX_STEPS * R.F32 + np.abs(dx64) * u * 1.01 + t)


@pytest.mark.parametrize("cols", [256, 777])
def test_odd_values(gsess, cols):
    """A NaN or an infinity spoils its own row only; a row of zeros norms to zeros; eps 0 on it gives NaN (0 / 0)."""
    x = np.random.default_rng(1).standard_normal((6, cols)).astype(np.float32)
    x[1, 3], x[3, cols - 1], x[4] = np.nan, np.inf, 0.0
    _, want = R.rmsnorm(x.astype(np.float64), None, None, 1e-6)
    got = gsess.rmsnorm(L.F32, x)
    R.close(got, want, np.abs(np.nan_to_num(want)) * Y_STEPS * R.F32)
    assert not got[4].any()
    assert np.isnan(gsess.rmsnorm(L.F32, x, eps=0.0)[4]).all()
    q, scales = gsess.rmsnorm(L.F32, x, quant=True, group=64)
    assert np.isnan(scales[1]).all() and (q[1] & 127 == 127).all() and np.isfinite(scales[[0, 2, 4, 5]]).all()


@pytest.mark.parametrize("dtype", R.DTYPES, ids=R.NAMES.get)
@pytest.mark.parametrize("cols", [2048, 333])
def test_outputs_in_place_of_inputs(gsess, dtype, cols):
    """The residual stream updated in its own buffer, y over x; dx over dy."""
    rng = np.random.default_rng(cols)
    rows = 70
    x, r, w = data(rng, (rows, cols), dtype), data(rng, (rows, cols), dtype, 2.0), data(rng, (cols,), dtype, 0.2, 1.0)
    h, y = gsess.rmsnorm(dtype, x, r, w)
    dx, dw = gsess.rmsnorm_bwd(dtype, h, x, w, r)
    pool, dev = gsess.pool, gsess.device
    bx, br, bw, bh, bdw = (pool.upload(a) for a in (x, r, w, h, np.zeros_like(w)))
    prog = dev.create_program(B.rmsnorm_desc(dtype, rows, cols, has_residual=True, has_weight=True))
    dev.launch(prog, [bx, br, bw, br, bx])
    assert np.array_equal(pool.download(br, h.shape, h.dtype), h) and np.array_equal(pool.download(bx, y.shape, y.dtype), y)
    dev.release(prog)
    bd, bq = pool.upload(x), pool.upload(r)
    prog = dev.create_program(B.rmsnorm_desc(dtype, rows, cols, has_weight=True, backward=True, has_dh=True))
    dev.launch(prog, [bh, bd, bw, bq, bd, bdw])
    assert np.array_equal(pool.download(bd, dx.shape, dx.dtype), dx) and np.array_equal(pool.download(bdw, dw.shape, dw.dtype), dw)
    dev.release(prog)
    for b in (bx, br, bw, bh, bdw, bd, bq):
        pool.deallocate(b)
    dev.check_guards()
