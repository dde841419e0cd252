"""The tolerance of the Muon step on the CPU: the kernels' arithmetic as tests/muon_model.py restates it keeps well inside it, and
a product that leaves out the low half of one operand does not."""
import numpy as np
import pytest

from tests import muon_model as M

SHAPES = [(128, 784), (48, 130), (300, 77), (130, 129), (100, 1500)]


def gradient(shape):
    rng = np.random.default_rng(shape[0])
    k = max(1, min(shape) // 16)
    return rng.standard_normal((shape[0], k)) @ rng.standard_normal((k, shape[1])) / np.sqrt(k) + rng.standard_normal(shape)


@pytest.mark.parametrize("shape", SHAPES)
def test_two_parts_stay_inside(shape):
    u = gradient(shape)
    want = M.exact(u)
    single, pair = M.single_part_error(u, want), float(np.linalg.norm(M.direction(u, 2) - want))
    assert 4 * pair <= single * M.TWO_PARTS, (pair, single)
    assert single <= 3e-3 * np.linalg.norm(want)


@pytest.mark.parametrize("which", range(3), ids=["gram", "polynomial", "result"])
@pytest.mark.parametrize("pair", [(1, 0), (0, 1)], ids=["left", "right"])
def test_a_dropped_low_half_is_seen(which, pair):
    u = gradient((128, 400))
    want = M.exact(u)
    dropped = [()] * 3
    dropped[which] = (pair,)
    wrong = float(np.linalg.norm(M.direction(u, 2, dropped=dropped) - want))
    assert wrong > 1.5 * M.single_part_error(u, want) * M.TWO_PARTS


def test_parts_and_sums():
    x = np.random.default_rng(0).standard_normal(1000) * 0.05
    one, two = M.parts(x, 1), M.parts(x, 2)
    assert np.abs(one[0] - x).max() <= np.abs(x).max() * 2.0 ** -11
    assert np.all(np.abs(sum(two) - x) <= np.abs(x) * 2.0 ** -21 + 2.0 ** -35)
    t = M.truncated(x)
    assert np.all(np.abs(t) <= np.abs(x)) and np.all(np.abs(t - x) <= np.abs(x) * 2.0 ** -23) and np.array_equal(M.truncated(t), t)
