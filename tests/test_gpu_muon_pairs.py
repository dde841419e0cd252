"""Muon's products on CTA pairs: updates queued back to back, so that one launch's CTAs take the places of the one before as they
leave, give the same bits every time and leave the device's status clear."""
import numpy as np
import pytest

from tests import operators_ref as R
from zyx_b200 import _lib as L
from zyx_b200 import backend as B

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gsess():
    from zyx_b200 import build
    from zyx_b200.ops import Session
    build.build()
    s = Session(device_ids=[0], debug=2, round_nearest=True)
    yield s
    s.close()


# 148 SMs: the symmetric products of six 1024 x 1024 take pairs with either number of parts, so does the last product of 1024 x 4096
# with two
@pytest.mark.parametrize("dtype", [L.F32, L.BF16], ids=R.NAMES.get)
@pytest.mark.parametrize("shapes", [[(1024, 1024)] * 6, [(1024, 4096)]], ids=["square", "wide"])
def test_updates_back_to_back(gsess, dtype, shapes):
    rng = np.random.default_rng(len(shapes))
    pool, dev = gsess.pool, gsess.device
    grads = [pool.upload(R.store(rng.standard_normal(s), dtype)) for s in shapes]
    sets = [[pool.upload(np.zeros(s, R.NP[dtype])) for s in shapes] for _ in range(12)]
    prog = dev.create_program(B.muon_desc(dtype, shapes, lr=1.0, momentum=0.0))
    for ps in sets:
        dev.launch(prog, ps + grads)
    got = [[pool.download(p, s, R.NP[dtype]) for p, s in zip(ps, shapes)] for ps in sets]
    assert dev.status() == 0
    dev.check_guards()
    for ps in got[1:]:
        assert all(np.array_equal(a, b) for a, b in zip(ps, got[0]))
    for p in got[0]:              # five steps take a broad spectrum near 1: the mean square of its singular values is that of p's norm
        assert 0.5 < np.linalg.norm(R.value(p, dtype)) / np.sqrt(min(p.shape)) < 1.25
    dev.release(prog)
    for b in grads + [b for ps in sets for b in ps]:
        pool.deallocate(b)
