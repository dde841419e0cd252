"""The Muon step itself (p = 0, lr = 1, no decay, no momentum) against 64 bits, in the Frobenius norm.

Tolerances come from the host's restatement of the arithmetic (muon_model.py; test_muon_model.py holds them against it): twice the
error of operands held as one f16 each for 16-bit matrices, a sixteenth of it for f32 ones, which hold them as two.  On top the
store into p: one rounding of each element."""
import numpy as np
import pytest

from tests import muon_model as M
from tests import operators_ref as R
from zyx_b200 import _lib as L

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gsess():
    from zyx_b200 import build
    from zyx_b200.ops import Session
    build.build()
    s = Session(device_ids=[0], debug=2, round_nearest=True)
    yield s
    s.close()


def gradient(rng, shape, dtype, scale=1.0):
    k = max(1, min(shape) // 16)
    g = rng.standard_normal((shape[0], k)) @ rng.standard_normal((k, shape[1])) / np.sqrt(k) + rng.standard_normal(shape)
    return R.store(g * scale, dtype)


def check(sess, dtype, shapes, scale=1.0, eps=0.0, **kw):
    rng = np.random.default_rng(shapes[0][0] * 29 + shapes[0][1])
    ts = [[np.zeros(s, R.NP[dtype]), gradient(rng, s, dtype, scale)] for s in shapes]
    sess.muon_step(dict(lr=1.0, momentum=0.0, eps=eps, **kw), dtype, ts)
    seen = {}
    for (p, g), shape in zip(ts, shapes):
        key = g.tobytes()
        if key not in seen:
            u = R.value(g, dtype)
            want = M.exact(u, eps=eps or 1e-7)
            seen[key] = want, M.single_part_error(u, want, eps=eps or 1e-7)
        want, single = seen[key]
        factor = R.adjust(L.MUON_ADJUST_RATIO, *shape)
        got = -R.value(p, dtype) / factor
        store = R.unit(dtype, True) * np.linalg.norm(want) + R.tiny(dtype, True) / factor * np.sqrt(want.size)
        off = np.linalg.norm(got - want)
        assert off <= single * (M.TWO_PARTS if dtype == L.F32 else M.ONE_PART) + store, (shape, off / single, single, store)


# one launch (up to 128 rows or columns), products with and without a split contraction, single CTAs and pairs
@pytest.mark.parametrize("dtype", R.DTYPES, ids=R.NAMES.get)
@pytest.mark.parametrize("shape", [(1, 4000), (16, 16), (48, 130), (128, 784), (784, 128), (128, 2048), (4096, 77), (130, 129), (129, 4100), (300, 77), (513, 260),
                                   (640, 640), (256, 1030), (2500, 200), (1024, 4096)])
def test_step(gsess, dtype, shape):
    check(gsess, dtype, [shape])


@pytest.mark.parametrize("dtype", R.DTYPES, ids=R.NAMES.get)
def test_step_of_several(gsess, dtype):
    check(gsess, dtype, [(1024, 1024)] * 6)
    check(gsess, dtype, [(64, 200), (200, 64), (64, 200), (30, 40)])


@pytest.mark.parametrize("dtype", [L.F32, L.BF16], ids=R.NAMES.get)
@pytest.mark.parametrize("shape", [(40, 72), (72, 40), (300, 260), (260, 300), (300, 261)])
@pytest.mark.parametrize("scale,eps", [(1e25, 0.0), (2e37, 0.0), (1e-3, 0.0), (1e-20, 1e-30), (1e-30, 1e-30)])
def test_large_and_small_gradients_are_normed_like_others(gsess, dtype, shape, scale, eps):
    """The norm of the gradients of 2e37 lies outside f32."""
    check(gsess, dtype, [shape], scale=scale, eps=eps)


@pytest.mark.parametrize("dtype", [L.F32, L.BF16], ids=R.NAMES.get)
@pytest.mark.parametrize("shape", [(40, 72), (300, 260)])
def test_a_gradient_far_below_eps_leaves_the_decay_only(gsess, dtype, shape):
    """1e-30 under the default eps of 1e-7: the direction is 1e-21 of a unit one, the step less than any rounding of p."""
    rng = np.random.default_rng(5)
    p = R.store(rng.standard_normal(shape), dtype)
    t = [p.copy(), gradient(rng, shape, dtype, 1e-30)]
    gsess.muon_step(dict(lr=0.5, weight_decay=0.125, momentum=0.0), dtype, [t])
    want = R.value(p, dtype) * (1 - 0.5 * 0.125)
    R.close(R.value(t[0], dtype), want, np.abs(want) * (R.unit(dtype, True) + 2 * R.F32) * 1.01 + R.tiny(dtype, True))
