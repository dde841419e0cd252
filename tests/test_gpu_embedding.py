"""Embedding lookup and the gradient of its table against 64-bit forms.

Tolerances: the lookup is one product and one store.  A gradient of k terms of magnitudes that add up to S is off by at most
(k + 1) half steps of f32 of S for its sums and the scale, and one store.
"""
import numpy as np
import pytest

from tests import operators_ref as R
from zyx_b200 import _lib as L
from zyx_b200 import backend as B

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", params=[True, False], ids=["nearest", "truncate"])
def gsess(request):
    from zyx_b200 import build
    from zyx_b200.ops import Session
    build.build()
    s = Session(device_ids=[0], debug=2, round_nearest=request.param)
    s.nearest = request.param
    yield s
    s.close()


def data(rng, shape, dtype, scale=1.0):
    return R.store(rng.standard_normal(shape) * scale, dtype)


def some_ids(rng, n, vocab, kind, id_dtype=np.int32):
    if kind == "uniform":
        ids = rng.integers(0, vocab, n)
    elif kind == "one":
        ids = np.full(n, vocab // 2)
    elif kind == "frequent":      # words by rank, scattered
        ids = rng.permutation(vocab)[np.minimum(vocab - 1, np.exp(rng.random(n) * np.log(vocab + 1)).astype(np.int64) - 1)]
    else:                         # "padded": outside numbers of every sort among the others
        ids = rng.integers(0, vocab, n)
        odd = np.array([-1, -100, vocab, vocab + 7, np.iinfo(id_dtype).min, np.iinfo(id_dtype).max])
        at = rng.random(n) < 0.4
        ids[at] = rng.choice(odd, int(at.sum()))
    return ids.astype(id_dtype)


SHAPES = [(1, 1, 1), (1, 5, 8), (8, 3000, 2048), (3, 7, 5), (130, 50, 64), (1000, 333, 100), (513, 4000, 777), (77, 11, 2050), (5, 3, 4098)]


@pytest.mark.parametrize("dtype", R.DTYPES, ids=R.NAMES.get)
@pytest.mark.parametrize("tokens,vocab,dim", SHAPES)
def test_lookup(gsess, dtype, tokens, vocab, dim):
    rng = np.random.default_rng(tokens + vocab + dim)
    table = data(rng, (vocab, dim), dtype)
    for id_dtype in (np.int32, np.int64):
        ids = some_ids(rng, tokens, vocab, "padded", id_dtype)
        got = gsess.embedding(dtype, ids, table)
        met = (ids >= 0) & (ids < vocab)
        want = np.zeros_like(got)
        want[met] = table[ids[met]]
        assert np.array_equal(got, want)                      # scale 1: the table's bits
    got = R.value(gsess.embedding(dtype, ids, table, scale=22.6), dtype)
    want = R.embedding(ids, R.value(table, dtype), float(np.float32(22.6)))
    R.close(got, want, np.abs(want) * (R.F32 * (1 + 2 ** -20) + R.unit(dtype, gsess.nearest)) + R.tiny(dtype, gsess.nearest))


def test_lookup_copies_what_the_table_holds(gsess):
    """NaN payloads, infinities and subnormals pass through a lookup without scale."""
    for dtype, bits in ((L.BF16, [0x7fc1, 0xff80, 0x0001, 0x8000]), (L.F16, [0x7e01, 0x7c00, 0x0001, 0x8001])):
        table = np.array(bits * 8, np.uint16).reshape(4, 8)
        ids = np.array([3, 0, 2, 2], np.int32)
        assert np.array_equal(gsess.embedding(dtype, ids, table), table[ids])


@pytest.mark.parametrize("dtype", R.DTYPES, ids=R.NAMES.get)
@pytest.mark.parametrize("kind", ["uniform", "one", "frequent", "padded"])
@pytest.mark.parametrize("tokens,vocab,dim", SHAPES + [(2500, 1500, 33), (4100, 150000, 16)])
def test_gradient(gsess, dtype, kind, tokens, vocab, dim):
    rng = np.random.default_rng(tokens * 3 + vocab + dim)
    ids = some_ids(rng, tokens, vocab, kind, np.int64 if dim % 2 else np.int32)
    dout = data(rng, (tokens, dim), dtype)
    scale = 1.0 if dim % 3 else 5.65
    want, mags, terms = R.embedding_bwd(ids, R.value(dout, dtype), vocab, float(np.float32(scale)))
    got = gsess.embedding_bwd(dtype, ids, dout, vocab, scale=scale)
    tol = (terms + 1) * R.F32 * mags + np.abs(want) * R.unit(dtype, gsess.nearest) * (1 + 2 ** -10) + R.tiny(dtype, gsess.nearest)
    R.close(R.value(got, dtype), want, tol)
    absent = (terms == 0).ravel()
    assert not R.value(got, dtype)[absent].any()
    again = gsess.embedding_bwd(dtype, ids, dout, vocab, scale=scale)
    assert np.array_equal(got, again)                         # the order of the sums depends on ids alone
    before = data(rng, (vocab, dim), dtype)
    got = gsess.embedding_bwd(dtype, ids, dout, vocab, scale=scale, accumulate_into=before)
    old = R.value(before, dtype)
    tol = (terms + 2) * R.F32 * (mags + np.abs(old)) + np.abs(want + old) * R.unit(dtype, gsess.nearest) * (1 + 2 ** -10) + R.tiny(dtype, gsess.nearest)
    R.close(R.value(got, dtype)[~absent], (want + old)[~absent], tol[~absent])
    assert np.array_equal(got[absent], before[absent])        # untouched


def test_gradient_against_differences(gsess):
    """<dtable, d> is the change of <dout, lookup(table)> along d: the lookup is linear, so the difference is the derivative."""
    rng = np.random.default_rng(5)
    tokens, vocab, dim = 300, 40, 24
    ids = some_ids(rng, tokens, vocab, "padded")
    table, d, dout = (rng.standard_normal(s).astype(np.float32) for s in ((vocab, dim), (vocab, dim), (tokens, dim)))
    up, down = gsess.embedding(L.F32, ids, table + d, scale=3.0), gsess.embedding(L.F32, ids, table - d, scale=3.0)
    change = float((dout.astype(np.float64) * (up.astype(np.float64) - down)).sum()) / 2
    grad = gsess.embedding_bwd(L.F32, ids, dout, vocab, scale=3.0).astype(np.float64)
    # each looked-up value is off by at most two half steps of its size (the sum table +- d, the product)
    size = float((np.abs(dout) * 3.0 * R.embedding(ids, np.abs(table) + np.abs(d), 1.0)).sum())
    assert abs(change - float((grad * d).sum())) <= size * 2 ** -20


@pytest.mark.parametrize("dtype", R.DTYPES, ids=R.NAMES.get)
def test_row_pitches_leave_the_space_between_rows(gsess, dtype):
    rng = np.random.default_rng(9)
    tokens, vocab, dim, ldt, ldo = 70, 45, 24, 40, 31
    ids = some_ids(rng, tokens, vocab, "padded")
    table = data(rng, (vocab, ldt), dtype)
    out0 = data(rng, (tokens, ldo), dtype)
    d = B.embedding_desc(dtype, tokens, vocab, dim, ld_table=ldt, ld_out=ldo)
    got = gsess.run(d, [ids, table], [((tokens, ldo), R.NP[dtype])], out_init=out0)[0]
    met = (ids >= 0) & (ids < vocab)
    want = out0.copy()
    want[:, :dim] = 0
    want[met, :dim] = table[ids[met], :dim]
    assert np.array_equal(got, want)
    dtable0 = data(rng, (vocab, ldt), dtype)
    d = B.embedding_desc(dtype, tokens, vocab, dim, ld_table=ldt, ld_out=ldo, backward=True)
    got = gsess.run(d, [ids, out0], [((vocab, ldt), R.NP[dtype])], out_init=dtable0)[0]
    assert np.array_equal(got[:, dim:], dtable0[:, dim:])
    want, mags, terms = R.embedding_bwd(ids, R.value(out0, dtype)[:, :dim], vocab)
    R.close(R.value(got, dtype)[:, :dim], want, (terms + 1) * R.F32 * mags + np.abs(want) * R.unit(dtype, gsess.nearest) * 1.01 + R.tiny(dtype, gsess.nearest))


def test_refusals_on_a_device(gsess):
    dev, pool = gsess.device, gsess.pool
    for kw in (dict(dim=0), dict(tokens=0), dict(vocab=0), dict(id_dtype=L.U8), dict(ld_out=3), dict(accumulate=True)):
        args = dict(tokens=4, vocab=4, dim=8)
        args.update(kw)
        with pytest.raises(Exception) as e:
            dev.create_program(B.embedding_desc(L.F32, **args))
        assert e.value.status_name == "KernelCompilation" and "embedding" in e.value.context
    prog = dev.create_program(B.embedding_desc(L.F32, 4, 4, 8))
    bufs = [pool.allocate(n)[0] for n in (16, 128, 128, 64)]
    with pytest.raises(Exception, match="out too small"):
        dev.launch(prog, [bufs[0], bufs[1], bufs[3]])
    with pytest.raises(Exception, match="of its own"):
        dev.launch(prog, [bufs[0], bufs[1], bufs[1]])
    with pytest.raises(Exception, match="expected args"):
        dev.launch(prog, bufs[:2])
    for b in bufs:
        pool.deallocate(b)
    dev.release(prog)
