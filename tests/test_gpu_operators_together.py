"""Embedding, RMS norm, the matmul and Muon as a training step uses them, on buffers that stay on the device; device memory of
another library as pool buffers; offsets beyond 32 bits.

Every stage of the step is held against its 64-bit form on the inputs it really had (read back from the device), with the
tolerances that the stages' own tests derive."""
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


class Step:
    """embed -> + residual, norm -> y W^T;  given dz and the stream's gradient: dW, dy, norm's adjoint, table gradient, Muon on W."""

    def __init__(self, s, dtype, tokens, vocab, dim, out, seed):
        self.s, self.dtype, self.shape = s, dtype, (tokens, vocab, dim, out)
        rng = np.random.default_rng(seed)
        ids = rng.integers(0, vocab, tokens).astype(np.int32)
        ids[-3:] = -1
        put = lambda *shape, scale=1.0, mean=0.0: R.store(rng.standard_normal(shape) * scale + mean, dtype)     # noqa: E731
        self.host = dict(ids=ids, table=put(vocab, dim, scale=0.02), stream=put(tokens, dim), gain=put(dim, scale=0.1, mean=1.0), w=put(out, dim, scale=0.05),
                         dz=put(tokens, out, scale=0.1), dstream=put(tokens, dim, scale=0.1), buf=np.zeros((out, dim), R.NP[dtype]))
        blank = dict(x=(tokens, dim), h=(tokens, dim), y=(tokens, dim), z=(tokens, out), dw=(out, dim), dy=(tokens, dim), dx=(tokens, dim), dgain=(dim,), dtable=(vocab, dim))
        self.host.update({k: np.zeros(v, R.NP[dtype]) for k, v in blank.items()})
        self.bufs = {k: s.pool.upload(v) for k, v in self.host.items()}
        t, v, d, o = tokens, vocab, dim, out
        mk = s.device.create_program
        self.plan = [
            (mk(B.embedding_desc(dtype, t, v, d, scale=float(d) ** 0.5)), "ids table x"),
            (mk(B.rmsnorm_desc(dtype, t, d, has_residual=True, has_weight=True)), "x stream gain h y"),
            (mk(B.gemm_desc(dtype, t, o, d, trans_b=True)), "y w z"),
            (mk(B.gemm_desc(dtype, o, d, t, trans_a=True)), "dz y dw"),
            (mk(B.gemm_desc(dtype, t, d, o)), "dz w dy"),
            (mk(B.rmsnorm_desc(dtype, t, d, has_weight=True, backward=True, has_dh=True)), "h dy gain dstream dx dgain"),
            (mk(B.embedding_desc(dtype, t, v, d, scale=float(d) ** 0.5, backward=True)), "ids dx dtable"),
            (mk(B.muon_desc(dtype, [(o, d)], lr=0.02, weight_decay=0.01)), "w dw buf"),
        ]

    def launch(self, upto=None):
        for prog, names in self.plan[:upto]:
            self.s.device.launch(prog, [self.bufs[n] for n in names.split()])

    def read(self):
        return {k: self.s.pool.download(self.bufs[k], v.shape, v.dtype) for k, v in self.host.items()}

    def close(self):
        for prog, _ in self.plan:
            self.s.device.release(prog)
        for b in self.bufs.values():
            self.s.pool.deallocate(b)


@pytest.mark.parametrize("dtype", R.DTYPES, ids=R.NAMES.get)
@pytest.mark.parametrize("shape", [(96, 50, 64, 128), (300, 1000, 136, 200)])
def test_a_training_step(gsess, dtype, shape):
    step = Step(gsess, dtype, *shape, seed=1)
    tokens, vocab, dim, out = shape
    u, tiny = R.unit(dtype, True), R.tiny(dtype, True)
    before = step.read()
    step.launch()
    got = step.read()
    v = {k: R.value(a, dtype) for k, a in got.items() if k != "ids"}
    scale = float(np.float32(float(dim) ** 0.5))
    want = R.embedding(got["ids"], R.value(before["table"], dtype), scale)
    R.close(v["x"], want, np.abs(want) * (u + 2 * R.F32) + tiny)
    h, y = R.rmsnorm(v["x"], v["stream"], v["gain"], float(np.float32(1e-6)))
    R.close(v["h"], h, np.abs(h) * (u + R.F32) * 1.01 + tiny)
    R.close(v["y"], y, np.abs(y) * (u + 40 * R.F32) * 1.01 + tiny)
    dx, dgain, size, gsize = R.rmsnorm_bwd(v["h"], v["dy"], v["gain"], v["dstream"], float(np.float32(1e-6)))
    R.close(v["dx"], dx, size * 120 * R.F32 + np.abs(dx) * u * 1.01 + tiny)
    R.close(v["dgain"], dgain, gsize * (tokens + 40) * R.F32 + np.abs(dgain) * u * 1.01 + tiny)
    total, mags, terms = R.embedding_bwd(got["ids"], v["dx"], vocab, scale)
    R.close(v["dtable"], total, (terms + 2) * R.F32 * mags + np.abs(total) * u * 1.01 + tiny)
    # W's own products are the matmul's business; its step is Muon's: buf = dW, X from (1 + mu) dW
    mu = float(np.float32(0.95))
    R.close(v["buf"], v["dw"], np.abs(v["dw"]) * (u + 2 * R.F32) + tiny)
    x, err = R.orthogonalise(v["dw"] + mu * v["buf"], rounding=2.0 ** -19 if dtype == L.F32 else 1.5 * 2.0 ** -11)
    lr = 0.02 * R.adjust(0, out, dim)
    p0 = R.value(before["w"], dtype)
    want = p0 * (1 - 0.02 * 0.01) - lr * x
    over = np.maximum(np.abs(v["w"] - want) - (np.abs(want) * u * 1.01 + (np.abs(p0) + lr * np.abs(x)) * 4 * R.F32 + tiny), 0)
    assert np.linalg.norm(over) <= lr * err
    gsess.device.check_guards()
    assert gsess.device.status() == 0
    step.close()


def test_replayed_steps_and_two_steps_at_once(gsess):
    """Three steps launched one by one, as a captured graph, and interleaved launch by launch with another step's: the same bits.
    (All of them share the context's scratch memory.)"""
    shape = (200, 333, 96, 160)
    results = []
    for how in ("plain", "graph", "interleaved", "two graphs"):
        a, b = Step(gsess, L.BF16, *shape, seed=2), Step(gsess, L.BF16, 130, 70, 200, 48, seed=3)
        dev, graphs = gsess.device, []
        if "graph" in how:
            for st in (a, b) if how == "two graphs" else (a,):
                dev.capture_begin()
                st.launch()
                graphs.append(dev.capture_end())
        for _ in range(3):
            if how == "plain":
                a.launch()
            elif graphs:
                for g in graphs:
                    dev.graph_launch(g)
            else:
                for (pa, na), (pb, nb) in zip(a.plan, b.plan):
                    dev.launch(pa, [a.bufs[n] for n in na.split()])
                    dev.launch(pb, [b.bufs[n] for n in nb.split()])
        results.append(a.read())
        for g in graphs:
            dev.graph_release(g)
        a.close()
        b.close()
    for r in results[1:]:
        for k in results[0]:
            assert np.array_equal(r[k], results[0][k]), k
    gsess.device.check_guards()


def test_a_new_program_after_a_released_one_has_memory_of_its_own(gsess):
    """Muon's workspace goes back to the pool with its program, behind the launches already queued."""
    rng = np.random.default_rng(7)
    g = R.store(rng.standard_normal((300, 260)), L.F32)
    want = None
    for _ in range(4):
        t = [np.zeros((300, 260), np.float32), g]
        bufs = [gsess.pool.upload(a) for a in t]
        prog = gsess.device.create_program(B.muon_desc(L.F32, [(300, 260)], lr=1.0, momentum=0.0))
        gsess.device.launch(prog, bufs)
        gsess.device.release(prog)
        other = gsess.pool.allocate(4 << 20)[0]
        gsess.pool.memset(other, 0xff, 4 << 20)
        got = gsess.pool.download(bufs[0], (300, 260), np.float32)
        want = got if want is None else want
        assert np.array_equal(got, want) and np.isfinite(got).all()
        for b in bufs + [other]:
            gsess.pool.deallocate(b)


# ---- memory of another library --------------------------------------------------------------------------------------------------
def test_programs_on_imported_memory(gsess):
    torch = pytest.importorskip("torch")
    table = torch.randn(50, 64, device="cuda")
    ids = torch.randint(0, 50, (33,), device="cuda", dtype=torch.int32)
    out = torch.zeros(33, 64, device="cuda")
    torch.cuda.synchronize()
    pool, dev = gsess.pool, gsess.device
    bufs = [pool.import_device(t.data_ptr(), t.numel() * t.element_size()) for t in (ids, table, out)]
    assert pool.buffer_bytes(bufs[1]) == 50 * 64 * 4
    prog = dev.create_program(B.embedding_desc(L.F32, 33, 50, 64))
    dev.launch(prog, bufs)
    dev.sync()
    assert torch.equal(out, table[ids.long()])
    assert np.array_equal(pool.download(bufs[2], (33, 64), np.float32), out.cpu().numpy())        # copies work on them too
    view = pool.view(bufs[1], 256, 256)
    assert np.array_equal(pool.download(view, (64,), np.float32), table[1].cpu().numpy())
    pool.deallocate(view)
    for b in bufs:
        pool.deallocate(b)
    assert torch.equal(out, table[ids.long()])                # only the ids are gone
    with pytest.raises(Exception, match="not a pool buffer"):
        dev.launch(prog, bufs)
    dev.release(prog)


def test_import_refusals(gsess):
    torch = pytest.importorskip("torch")
    pool = gsess.pool
    t = torch.zeros(1 << 16, device="cuda")
    for args, text in (((0, 16), "null"), ((t.data_ptr(), 0), "no bytes"), ((t.data_ptr() + 16, 16), "256"), ((t.data_ptr(), 1 << 44), "exceeds the allocation")):
        with pytest.raises(Exception, match=text):
            pool.import_device(*args)
    host = np.zeros(4096, np.uint8)
    with pytest.raises(Exception, match="not memory of this device"):
        pool.import_device((host.ctypes.data + 255) // 256 * 256, 16)
    buf = pool.import_device(t.data_ptr(), 64)
    with pytest.raises(Exception, match="exceeds"):
        pool.host_to_pool(np.zeros(65, np.uint8), buf)
    pool.deallocate(buf)


# ---- offsets beyond 32 bits -----------------------------------------------------------------------------------------------------
def test_a_table_of_more_than_four_gigaelements(gsess):
    vocab, dim = (1 << 21) + 5, 2048                          # 2^32 + 10240 elements of bf16
    pool, dev = gsess.pool, gsess.device
    nbytes = vocab * dim * 2
    if pool.free_bytes() < 2 * nbytes:
        pytest.skip("needs 9 GB")
    table = pool.allocate(nbytes)[0]
    pool.memset(table, 0, nbytes)
    rng = np.random.default_rng(0)
    row = R.store(rng.standard_normal(dim), L.BF16)
    pool.sync_events([pool.host_to_pool(row, table, dst_offset=(vocab - 1) * dim * 2)])
    ids = np.array([vocab - 1, 0, vocab - 2, vocab - 1, vocab], np.int32)
    bi, bo = pool.upload(ids), pool.allocate(5 * dim * 2)[0]
    prog = dev.create_program(B.embedding_desc(L.BF16, 5, vocab, dim))
    dev.launch(prog, [bi, table, bo])
    got = pool.download(bo, (5, dim), np.uint16)
    assert np.array_equal(got[[0, 3]], np.stack([row, row])) and not got[[1, 2, 4]].any()
    dev.release(prog)
    pool.memset(table, 0x55, nbytes)
    prog = dev.create_program(B.embedding_desc(L.BF16, 5, vocab, dim, backward=True))
    dev.launch(prog, [bi, bo, table])
    last = np.empty(dim, np.uint16)
    pool.pool_to_host(table, last, src_offset=(vocab - 1) * dim * 2)
    assert np.array_equal(R.value(last, L.BF16), 2 * R.value(row, L.BF16))
    for r in (0, 1, vocab // 2, vocab - 3, vocab - 2):
        pool.pool_to_host(table, last, src_offset=r * dim * 2)
        assert not last.any(), r
    dev.check_guards()
    dev.release(prog)
    for b in (table, bi, bo):
        pool.deallocate(b)


@pytest.mark.parametrize("pitch", [(1 << 32) + 8, (1 << 32) + 3])
def test_rows_more_than_four_gigaelements_apart(gsess, pitch):
    cols = 100
    pool, dev = gsess.pool, gsess.device
    nbytes = (pitch + cols) * 2
    if pool.free_bytes() < 3 * nbytes:
        pytest.skip("needs 26 GB")
    bx, by = pool.allocate(nbytes)[0], pool.allocate(nbytes)[0]
    rng = np.random.default_rng(0)
    x = R.store(rng.standard_normal((2, cols)), L.BF16)
    for r in range(2):
        pool.sync_events([pool.host_to_pool(x[r], bx, dst_offset=r * pitch * 2)])
    for kw, args in ((dict(), [bx, by]), (dict(backward=True), [bx, bx, by])):
        prog = dev.create_program(B.rmsnorm_desc(L.BF16, 2, cols, ld=pitch, **kw))
        dev.launch(prog, args)
        got = np.empty((2, cols), np.uint16)
        for r in range(2):
            pool.pool_to_host(by, got[r], src_offset=r * pitch * 2)
        v = R.value(x, L.BF16)
        if kw:
            want, _, size, _ = R.rmsnorm_bwd(v, v, None, None, 1e-6)
            R.close(R.value(got, L.BF16), want, size * 120 * R.F32 + np.abs(want) * 2.0 ** -8 * 1.01)
        else:
            want = R.rmsnorm(v, None, None, 1e-6)[1]
            R.close(R.value(got, L.BF16), want, np.abs(want) * (2.0 ** -8 + 40 * R.F32) * 1.01)
        dev.release(prog)
    dev.check_guards()
    pool.deallocate(bx)
    pool.deallocate(by)
