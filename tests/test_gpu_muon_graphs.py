"""A Muon program keeps its workspace while a graph that captured its launch lives: a replay never writes to memory of a new owner."""
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


def test_release_is_refused_while_a_graph_lives(gsess):
    pool, dev = gsess.pool, gsess.device
    shape = (300, 260)
    g = pool.upload(R.store(np.random.default_rng(0).standard_normal(shape), L.F32))
    p = pool.upload(np.zeros(shape, np.float32))
    prog = dev.create_program(B.muon_desc(L.F32, [shape], lr=1.0, momentum=0.0))
    other = dev.create_program(B.muon_desc(L.F32, [shape], lr=1.0, momentum=0.0))
    graphs = []
    for _ in range(2):
        dev.capture_begin()
        dev.launch(prog, [p, g])
        dev.launch(prog, [p, g])
        with pytest.raises(Exception, match="expected args"):
            dev.launch(other, [p])                        # refused: not part of the graph
        graphs.append(dev.capture_end())
    dev.release(other)
    for graph in graphs:
        with pytest.raises(Exception, match="release the graph first"):
            dev.release(prog)
        dev.graph_launch(graph)
        dev.graph_release(graph)
    dev.launch(prog, [p, g])
    dev.release(prog)
    block = pool.allocate(8 << 20)[0]                     # may be the workspace
    pool.memset(block, 0x5a, 8 << 20)
    got = pool.download(p, shape, np.float32)
    once = [[np.zeros(shape, np.float32), pool.download(g, shape, np.float32)]]
    gsess.muon_step(dict(lr=1.0, momentum=0.0), L.F32, once)
    x = once[0][0].astype(np.float64)
    R.close(got, 5 * x, np.abs(x) * 5 * 6 * R.F32)        # five equal steps, five roundings of the sum
    assert np.all(pool.download(block, (8 << 20,), np.uint8) == 0x5a)
    for b in (g, p, block):
        pool.deallocate(b)
    dev.check_guards()
