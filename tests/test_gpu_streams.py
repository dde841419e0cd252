"""Programs on a caller's stream (zyxb_use_stream): in order with another library's work on imported memory, without a
synchronisation anywhere; going back; what is refused."""
import numpy as np
import pytest

from zyx_b200 import _lib as L
from zyx_b200 import backend as B

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
TOKENS, VOCAB, DIM = 4096, 3000, 512
DELAY = 20_000_000          # clocks of a bounded device sleep, some 10 ms: what comes behind it has not run when the host goes on


@pytest.fixture(scope="module")
def gsess():
    from zyx_b200 import build
    from zyx_b200.ops import Session
    build.build()
    s = Session(device_ids=[0], debug=2, round_nearest=True)
    yield s
    s.close()


@pytest.mark.parametrize("side", [False, True], ids=["default stream", "side stream"])
def test_torch_before_and_after_without_a_wait(gsess, side):
    pool, dev = gsess.pool, gsess.device
    stream = torch.cuda.Stream() if side else torch.cuda.default_stream()
    source = torch.randn(VOCAB, DIM, device="cuda")
    ids = torch.randint(0, VOCAB, (TOKENS,), device="cuda", dtype=torch.int32)
    table, out = torch.zeros_like(source), torch.zeros(TOKENS, DIM, device="cuda")
    torch.cuda.synchronize()
    bufs = [pool.import_device(t.data_ptr(), t.numel() * t.element_size()) for t in (ids, table, out)]
    prog = dev.create_program(B.embedding_desc(L.F32, TOKENS, VOCAB, DIM))
    dev.use_stream(stream.cuda_stream)
    try:
        got = []
        with torch.cuda.stream(stream):
            for k in range(4):
                torch.cuda._sleep(DELAY)
                table.copy_(source).mul_(k + 1)             # late: behind the sleep
                dev.launch(prog, bufs)
                got.append(out.clone())
                torch.cuda._sleep(DELAY)
                out.fill_(-1.0)                             # written again while the host is far ahead
        torch.cuda.synchronize()
        for k, g in enumerate(got):
            assert torch.equal(g, source[ids.long()] * (k + 1)), k
    finally:
        dev.use_stream(None)
        for b in bufs:
            pool.deallocate(b)
        dev.release(prog)


def test_there_and_back_keeps_the_order(gsess):
    """The same buffer written on the own stream, on a caller's and on the own one again."""
    pool, dev = gsess.pool, gsess.device
    stream = torch.cuda.Stream()
    buf = pool.allocate(1 << 20)[0]
    n = 1 << 18
    prog = dev.create_program(B.eltwise_desc(L.EW_SCALE, L.F32, n, p0=2.0))
    pool.sync_events([pool.host_to_pool(np.ones(n, np.float32), buf)])
    for k in range(12):
        dev.use_stream(stream.cuda_stream if k % 3 == 0 else torch.cuda.default_stream().cuda_stream if k % 3 == 1 else None)
        if k % 3 == 0:
            with torch.cuda.stream(stream):
                torch.cuda._sleep(DELAY // 4)
        dev.launch(prog, [buf, buf])
    dev.use_stream(None)
    assert np.array_equal(pool.download(buf, (n,), np.float32), np.full(n, 4096, np.float32))
    dev.use_stream(stream.cuda_stream)                      # uploads, downloads and a captured launch on the caller's stream
    pool.host_to_pool(np.full(n, 3, np.float32), buf, want_event=False)
    dev.capture_begin()
    dev.launch(prog, [buf, buf])
    graph = dev.capture_end()
    dev.graph_launch(graph)
    dev.graph_launch(graph)
    assert np.array_equal(pool.download(buf, (n,), np.float32), np.full(n, 12, np.float32))
    dev.graph_release(graph)
    dev.use_stream(None)
    dev.release(prog)
    pool.deallocate(buf)
    dev.check_guards()


def test_refusals(gsess):
    dev = gsess.device
    with pytest.raises(Exception, match="per-thread"):
        dev.use_stream(2)                                   # cudaStreamPerThread
    dev.capture_begin()
    with pytest.raises(Exception, match="not allowed between"):
        dev.use_stream(0)
    dev.graph_release(dev.capture_end())
    dev.use_stream(1)                                       # cudaStreamLegacy, the default stream's other name
    with pytest.raises(Exception, match="cudaStreamBeginCapture"):
        dev.capture_begin()
    assert np.array_equal(gsess.eltwise(L.EW_SCALE, L.F32, np.ones(8, np.float32), p0=3.0), np.full(8, 3, np.float32))      # the refusal left nothing behind
    dev.use_stream(None)
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    x = torch.zeros(8, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
        x += 1
        with pytest.raises(Exception, match="being captured"):
            dev.use_stream(stream.cuda_stream)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(x, torch.ones_like(x))


def test_a_context_that_ends_leaves_the_stream_to_its_owner():
    from zyx_b200.ops import Session
    s = Session(device_ids=[0])
    stream = torch.cuda.Stream()
    s.device.use_stream(stream.cuda_stream)
    s.eltwise(L.EW_SCALE, L.F32, np.ones(8, np.float32), p0=3.0)
    s.close()
    with torch.cuda.stream(stream):
        x = torch.ones(8, device="cuda") * 2
    stream.synchronize()
    assert torch.equal(x, torch.full_like(x, 2))
