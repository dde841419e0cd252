"""The Muon program against a 64-bit form.

Tolerance of the orthogonalised step, in the Frobenius norm: operators_ref.orthogonalise carries a bound through the iteration on
its actual singular values.  What it is given per rounding: 16-bit matrices hold X, A and the polynomial as f16 (2^-11) under f32
sums whose truncation adds at most 2^-24 per product of 16 (2^-13 at 32768), so 2^-11 * 1.5; f32 matrices hold them as pairs of f16
(2^-22, and as much for the dropped product of the low halves), sums in f32 of at most 32768 / 16 products with rounding in both
directions: 2^-19.
"""
import numpy as np
import pytest

from tests import operators_ref as R
from zyx_b200 import _lib as L
from zyx_b200 import backend as B

pytestmark = pytest.mark.gpu
ROUNDING = {L.F32: 2.0 ** -19, L.BF16: 1.5 * 2.0 ** -11, L.F16: 1.5 * 2.0 ** -11}


@pytest.fixture(scope="module", params=[True, False], ids=["nearest", "truncate"])
def gsess(request):
    from zyx_b200 import build
    from zyx_b200.ops import Session
    build.build()
    s = Session(device_ids=[0], debug=2, round_nearest=request.param)
    s.nearest = request.param
    yield s
    s.close()


def gradient(rng, rows, cols, dtype, scale=1e-3):
    """a few strong directions over a broad floor"""
    k = max(1, min(rows, cols) // 16)
    g = rng.standard_normal((rows, k)) @ rng.standard_normal((k, cols)) / np.sqrt(k) + rng.standard_normal((rows, cols))
    return R.store(g * scale, dtype)


def check(sess, dtype, shapes, rng, lr=0.02, weight_decay=0.01, momentum=0.95, nesterov=True, steps=0, coefficients=(0.0, 0.0, 0.0), grad_scale=0.0,
          adjust=L.MUON_ADJUST_RATIO, p_scale=0.02, grads=None):
    ts = []
    for i, (r, c) in enumerate(shapes):
        t = [R.store(rng.standard_normal((r, c)) * p_scale, dtype), gradient(rng, r, c, dtype) if grads is None else grads[i]]
        if momentum:
            t.append(R.store(rng.standard_normal((r, c)) * 1e-3, dtype))
        ts.append(t)
    before = [[a.copy() for a in t] for t in ts]
    sess.muon_step(dict(lr=lr, weight_decay=weight_decay, momentum=momentum, nesterov=nesterov, steps=steps, coefficients=coefficients,
                        grad_scale=grad_scale, adjust=adjust), dtype, ts)
    u, tiny = R.unit(dtype, sess.nearest), R.tiny(dtype, sess.nearest)
    abc = tuple(float(np.float32(v)) for v in (coefficients if any(coefficients) else R.NS))
    for t, old, (r, c) in zip(ts, before, shapes):
        g = R.value(old[1], dtype) * (float(np.float32(grad_scale)) if grad_scale else 1.0)
        assert np.array_equal(t[1], old[1])
        if momentum:
            mu = float(np.float32(momentum))
            b64 = mu * R.value(old[2], dtype) + g
            R.close(R.value(t[2], dtype), b64, (np.abs(mu * R.value(old[2], dtype)) + np.abs(g)) * 3 * R.F32 + np.abs(b64) * u * 1.01 + tiny)
            buf = R.value(t[2], dtype)
            d = g + mu * buf if nesterov else buf
        else:
            d = g
        x, err = R.orthogonalise(d, steps or 5, abc, 1e-7, ROUNDING[dtype])
        step = lr * R.adjust(adjust, r, c)
        p0, got = R.value(old[0], dtype), R.value(t[0], dtype)
        want = p0 * (1 - lr * weight_decay) - step * x
        # per element: the store and three f32 roundings; over the matrix: the step's own error
        slack = np.abs(want) * u * 1.01 + (np.abs(p0) + step * np.abs(x)) * 4 * R.F32 + tiny
        over = np.maximum(np.abs(got - want) - slack, 0.0)
        assert np.linalg.norm(over) <= step * err + 1e-30, (r, c, np.linalg.norm(over) / step, err, np.linalg.norm(x))
    return ts


# up to 128 rows or columns: one launch, while X fits eight CTAs (2048 columns of f32, 4096 of 16-bit); the rest by products
SHAPES = [(1, 1), (1, 9), (7, 1), (5, 3), (16, 16), (33, 70), (128, 784), (10, 128), (128, 2048), (1999, 100), (2049, 128), (77, 4096), (4097, 33), (130, 129),
          (300, 77), (513, 260), (256, 1030), (640, 640), (129, 4100), (2500, 200), (384, 1537)]


@pytest.mark.parametrize("dtype", R.DTYPES, ids=R.NAMES.get)
@pytest.mark.parametrize("shape", SHAPES)
def test_update(gsess, dtype, shape):
    check(gsess, dtype, [shape], np.random.default_rng(shape[0] * 31 + shape[1]))


@pytest.mark.parametrize("dtype", R.DTYPES, ids=R.NAMES.get)
def test_the_step_alone_and_its_singular_values(gsess, dtype):
    """p = 0, lr = 1, no decay: the step itself.  Five steps of the default polynomial take every singular value of at least 0.01 of
    the norm into [0.65, 1.25]."""
    for shape in ((96, 200), (200, 96), (150, 150)):
        rng = np.random.default_rng(shape[0])
        q1, q2 = np.linalg.qr(rng.standard_normal((shape[0], 96)))[0], np.linalg.qr(rng.standard_normal((shape[1], 96)))[0]
        if min(shape) == 96:
            g = R.store(q1 @ np.diag(np.linspace(0.3, 1.0, 96)) @ q2.T, dtype)
            ts = check(gsess, dtype, [shape], rng, lr=1.0, weight_decay=0.0, momentum=0.0, p_scale=0.0, grads=[g])
            s = np.linalg.svd(R.value(ts[0][0], dtype) / R.adjust(0, *shape), compute_uv=False)
            assert s.min() > 0.6 and s.max() < 1.3
        else:
            check(gsess, dtype, [shape], rng, lr=1.0, weight_decay=0.0, momentum=0.0, p_scale=0.0)


@pytest.mark.parametrize("dtype", R.DTYPES, ids=R.NAMES.get)
@pytest.mark.parametrize("kw", [dict(momentum=0.0), dict(nesterov=False), dict(steps=1), dict(steps=9, coefficients=(1.5, -0.5, 0.0)),
                                dict(coefficients=(1.875, -1.25, 0.375)), dict(grad_scale=0.125), dict(adjust=L.MUON_ADJUST_RMS),
                                dict(weight_decay=0.0)], ids=str)
def test_options(gsess, dtype, kw):
    check(gsess, dtype, [(48, 130), (130, 48)], np.random.default_rng(8), **kw)


@pytest.mark.parametrize("dtype", R.DTYPES, ids=R.NAMES.get)
def test_many_matrices_of_mixed_shapes(gsess, dtype):
    """Equal shapes, their transposes, and others in between; more than one table of them."""
    shapes = [(64, 96), (64, 96), (96, 64), (10, 128), (64, 96), (96, 64), (33, 5)] + [(24, 40)] * 40
    check(gsess, dtype, shapes, np.random.default_rng(4))


@pytest.mark.parametrize("dtype", R.DTYPES, ids=R.NAMES.get)
@pytest.mark.parametrize("shape", [(330, 650), (328, 648)])
def test_more_tiles_than_a_launch_has_ctas(gsess, dtype, shape):
    """24 matrices of 66 tiles of 64 x 64 each, lying and standing: the CTAs that lay out X take several."""
    check(gsess, dtype, [shape, shape[::-1]] * 12, np.random.default_rng(12))


@pytest.mark.parametrize("dtype", R.DTYPES, ids=R.NAMES.get)
def test_zero_and_odd_gradients(gsess, dtype):
    """A zero gradient moves p by the decay only; tiny and huge ones are normed like others; a NaN stays in its own matrix."""
    rng = np.random.default_rng(2)
    r, c = 40, 72
    zero, good = R.store(np.zeros((r, c)), dtype), gradient(rng, r, c, dtype)
    nan = good.copy()
    nan[3, 5] = R.store(np.array([np.nan]), dtype)[0]
    ps = [R.store(rng.standard_normal((r, c)), dtype) for _ in range(3)]
    ts = [[p.copy(), g] for p, g in zip(ps, (zero, nan, good))]
    gsess.muon_step(dict(lr=0.5, weight_decay=0.125, momentum=0.0), dtype, ts)
    want = R.value(ps[0], dtype) * (1 - 0.5 * 0.125)
    R.close(R.value(ts[0][0], dtype), want, np.abs(want) * (R.unit(dtype, gsess.nearest) + 2 * R.F32) * 1.01 + R.tiny(dtype, gsess.nearest))
    assert np.isnan(R.value(ts[1][0], dtype)).all()
    alone = [[ps[2].copy(), good]]
    gsess.muon_step(dict(lr=0.5, weight_decay=0.125, momentum=0.0), dtype, alone)
    assert np.array_equal(alone[0][0], ts[2][0])
    if dtype != L.F16:
        for scale in (1e-30, 1e25):
            check(gsess, dtype, [(r, c)], rng, momentum=0.0, grads=[gradient(rng, r, c, dtype, scale)]) if scale > 1 else \
                gsess.muon_step(dict(lr=0.5, momentum=0.0), dtype, [[ps[0].copy(), gradient(rng, r, c, dtype, scale)]])


def test_repeated_steps_and_a_captured_launch(gsess):
    """The program has no step counter: launches captured into a graph and replayed equal launches made one by one."""
    rng = np.random.default_rng(6)
    pool, dev = gsess.pool, gsess.device
    r, c = 192, 320
    p, g, buf = (R.store(rng.standard_normal((r, c)) * 0.02, L.BF16) for _ in range(3))
    results = []
    for captured in (False, True):
        bufs = [pool.upload(a) for a in (p, g, buf)]
        prog = dev.create_program(B.muon_desc(L.BF16, [(r, c)], lr=0.02))
        if captured:
            dev.capture_begin()
            dev.launch(prog, bufs)
            with pytest.raises(Exception, match="not allowed between"):
                dev.create_program(B.muon_desc(L.BF16, [(r, c)], lr=0.02))
            with pytest.raises(Exception, match="not allowed between"):
                dev.release(prog)
            graph = dev.capture_end()
        for _ in range(3):
            dev.graph_launch(graph) if captured else dev.launch(prog, bufs)
        results.append([pool.download(bufs[0], p.shape, p.dtype), pool.download(bufs[2], p.shape, p.dtype)])
        if captured:
            dev.graph_release(graph)
        dev.release(prog)
        for b in bufs:
            pool.deallocate(b)
    assert all(np.array_equal(a, b) for a, b in zip(*results))
    dev.check_guards()
    assert dev.status() == 0
