"""The RMS norm and its adjoint where the rule that spreads a row over threads changes: widths between 2046 and 6145 columns with
few and with many rows.  Same 64-bit forms and tolerances as test_gpu_rmsnorm.py."""
import numpy as np
import pytest

from tests import operators_ref as R
from zyx_b200 import _lib as L

pytestmark = pytest.mark.gpu
Y_STEPS, DX_STEPS = 40, 120


@pytest.fixture(scope="module")
def gsess():
    from zyx_b200 import build
    from zyx_b200.ops import Session
    build.build()
    s = Session(device_ids=[0], debug=2, round_nearest=True)
    yield s
    s.close()


def data(rng, shape, dtype, scale=1.0, mean=0.0):
    return R.store(rng.standard_normal(shape) * scale + mean, dtype)


# a row is spread one vector per thread below 2048 vectors per SM: 148 SMs give 473 rows of 640 vectors, 394 of 768
SHAPES = [(r, c) for c in (2046, 2052, 2304, 2560, 2880, 3069, 3071, 3076) for r in (1, 64, 394)] + \
         [(473, 2560), (474, 2560), (590, 2052), (591, 2052), (7, 4097), (7, 6143), (7, 6145), (300, 6144)]


@pytest.mark.parametrize("rows,cols", SHAPES)
def test_adjoint_f32(gsess, rows, cols):
    rng = np.random.default_rng(rows * 13 + cols)
    h, dy, w, dh = data(rng, (rows, cols), L.F32, 2.0), data(rng, (rows, cols), L.F32), data(rng, (cols,), L.F32, 0.2, 1.0), data(rng, (rows, cols), L.F32)
    for weight, add in ((w, dh), (None, None)):
        dx64, dw64, size, dw_size = R.rmsnorm_bwd(*(None if a is None else a.astype(np.float64) for a in (h, dy, weight, add)), 1e-6)
        got = gsess.rmsnorm_bwd(L.F32, h, dy, weight, add)
        if weight is not None:
            got, dw = got
            R.close(dw, dw64, dw_size * (rows + Y_STEPS) * R.F32 + np.abs(dw64) * R.F32)
        R.close(got, dx64, size * DX_STEPS * R.F32 + np.abs(dx64) * R.F32)


@pytest.mark.parametrize("dtype", R.DTYPES, ids=R.NAMES.get)
@pytest.mark.parametrize("rows,cols", [(8, 2560), (394, 3071), (8, 4104), (8, 5120), (8, 6152), (600, 8190)])
def test_both_directions(gsess, dtype, rows, cols):
    rng = np.random.default_rng(rows * 17 + cols)
    x, dy, w = data(rng, (rows, cols), dtype, 2.0), data(rng, (rows, cols), dtype), data(rng, (cols,), dtype, 0.2, 1.0)
    u, t = R.unit(dtype, True), R.tiny(dtype, True)
    xv, dv, wv = (R.value(a, dtype) for a in (x, dy, w))
    y64 = R.rmsnorm(xv, None, wv, 1e-6)[1]
    R.close(R.value(gsess.rmsnorm(dtype, x, None, w), dtype), y64, np.abs(y64) * (Y_STEPS * R.F32 + u) * 1.01 + t)
    dx64, dw64, size, dw_size = R.rmsnorm_bwd(xv, dv, wv, None, 1e-6)
    dx, dw = gsess.rmsnorm_bwd(dtype, x, dy, w)
    R.close(R.value(dx, dtype), dx64, size * DX_STEPS * R.F32 + np.abs(dx64) * u * 1.01 + t)
    R.close(R.value(dw, dtype), dw64, dw_size * (rows + Y_STEPS) * R.F32 + np.abs(dw64) * u * 1.01 + t)
