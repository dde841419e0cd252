"""What the embedding, RMS norm and Muon programs refuse, on the CPU: at creation (KernelCompilation) and at launch, before anything
reaches a device (IncorrectKernelArg).  Addresses are made up; the checks run in a process without a GPU."""
import json
import os
import subprocess
import sys

import pytest

from zyx_b200 import _lib as L

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
E, EB = dict(dtype=L.F32, tokens=4, vocab=10, dim=8), dict(dtype=L.F32, tokens=4, vocab=10, dim=8, backward=True)
N, NB = dict(dtype=L.BF16, rows=4, cols=64), dict(dtype=L.BF16, rows=4, cols=64, backward=True, has_weight=True, has_dh=True)
M = dict(dtype=L.BF16, shapes=[[8, 16], [8, 16]], lr=0.1)
BIG = 1 << 20


def buf(*sizes):
    return [[(i + 1) << 24, s] for i, s in enumerate(sizes)]


CREATE = [
    ("embedding_desc", dict(E, dtype=L.I32), "dtype"), ("embedding_desc", dict(E, id_dtype=L.F32), "id_dtype"), ("embedding_desc", dict(E, tokens=0), "positive"),
    ("embedding_desc", dict(E, vocab=0), "positive"), ("embedding_desc", dict(E, dim=0), "positive"), ("embedding_desc", dict(E, tokens=1 << 31), "2^31"),
    ("embedding_desc", dict(E, dim=(1 << 20) + 1), "2^20"), ("embedding_desc", dict(E, ld_table=7), "pitch"), ("embedding_desc", dict(E, ld_out=7), "pitch"),
    ("embedding_desc", dict(E, ld_out=1 << 41), "pitch"), ("embedding_desc", dict(E, accumulate=True), "gradient"),
    ("embedding_desc", dict(EB, tokens=(1 << 24) + 1), "2^24"), ("embedding_desc", dict(EB, vocab=(1 << 24) + 1), "2^24"),
    ("rmsnorm_desc", dict(N, dtype=L.U8), "dtype"), ("rmsnorm_desc", dict(N, rows=0), "positive"), ("rmsnorm_desc", dict(N, cols=0), "positive"),
    ("rmsnorm_desc", dict(N, cols=16385), "16384"), ("rmsnorm_desc", dict(N, ld=63), "pitch"), ("rmsnorm_desc", dict(N, eps=-1.0), "eps"),
    ("rmsnorm_desc", dict(N, eps=float("nan")), "eps"), ("rmsnorm_desc", dict(N, group=64), "quant"), ("rmsnorm_desc", dict(N, quant=True, group=15), "16"),
    ("rmsnorm_desc", dict(N, has_dh=True), "backward"), ("rmsnorm_desc", dict(NB, quant=True), "forward"), ("rmsnorm_desc", dict(NB, has_residual=True), "forward"),
    ("muon_desc", dict(M, dtype=L.F64), "dtype"), ("muon_desc", dict(M, shapes=[]), "1 to 1024"), ("muon_desc", dict(M, shapes=[[0, 4]]), "extents"),
    ("muon_desc", dict(M, shapes=[[4, 32769]]), "extents"), ("muon_desc", dict(M, steps=33), "steps"), ("muon_desc", dict(M, steps=-1), "steps"),
    ("muon_desc", dict(M, eps=1e-31), "eps"), ("muon_desc", dict(M, eps=-1.0), "eps"), ("muon_desc", dict(M, adjust=2), "adjust"),
    ("muon_desc", dict(M, coefficients=[3.5, 0.0, 0.0]), "1.25"), ("muon_desc", dict(M, coefficients=[float("nan"), 0.0, 1.0]), "1.25"),
]
LAUNCH = [
    ("embedding_desc", E, buf(16, 320), "expected args"), ("embedding_desc", E, buf(15, 320, 128), "ids"), ("embedding_desc", E, buf(16, 319, 128), "table"),
    ("embedding_desc", E, buf(16, 320, 127), "out"), ("embedding_desc", dict(E, id_dtype=L.I64), buf(31, 320, 128), "ids"),
    ("embedding_desc", dict(E, ld_out=9), buf(16, 320, 139), "out"), ("embedding_desc", E, [[1 << 24, BIG], [2 << 24, BIG], [2 << 24, BIG]], "of its own"),
    ("embedding_desc", E, [[1 << 24, BIG], [2 << 24, BIG], [1 << 24, BIG]], "of its own"),
    ("embedding_desc", EB, buf(16, 127, 320), "dout"), ("embedding_desc", EB, buf(16, 128, 319), "dtable"),
    ("embedding_desc", EB, [[1 << 24, BIG], [2 << 24, BIG], [2 << 24, BIG]], "of its own"),
    # the last row's offset needs more than 64 bits of bytes
    ("embedding_desc", dict(E, tokens=(1 << 31) - 1, ld_out=1 << 40), buf(1 << 34, BIG, BIG), "out"),
    ("rmsnorm_desc", N, buf(512), "expected args"), ("rmsnorm_desc", N, buf(511, 512), "x too small"), ("rmsnorm_desc", N, buf(512, 511), "y too small"),
    ("rmsnorm_desc", dict(N, ld=65), buf(BIG, 517), "y too small"), ("rmsnorm_desc", dict(N, has_weight=True), buf(512, 127, 512), "weight"),
    ("rmsnorm_desc", dict(N, has_residual=True), buf(512, 511, 512, 512), "residual"), ("rmsnorm_desc", dict(N, has_residual=True), buf(512, 512, 511, 512), "h too small"),
    ("rmsnorm_desc", dict(N, has_residual=True), [[1 << 24, BIG], [2 << 24, BIG], [3 << 24, BIG], [3 << 24, BIG]], "different"),
    ("rmsnorm_desc", dict(N, has_weight=True), [[1 << 24, BIG], [2 << 24, BIG], [2 << 24, BIG]], "weight"),
    ("rmsnorm_desc", dict(N, quant=True, group=16), buf(512, 255, 64), "y too small"), ("rmsnorm_desc", dict(N, quant=True, group=16), buf(512, 256, 63), "scales"),
    ("rmsnorm_desc", dict(N, quant=True), [[1 << 24, BIG], [1 << 24, BIG], [3 << 24, BIG]], "of their own"),
    ("rmsnorm_desc", dict(N, quant=True), [[1 << 24, BIG], [2 << 24, BIG], [2 << 24, BIG]], "of their own"),
    ("rmsnorm_desc", NB, buf(512, 512, 128, 512, 512), "expected args"), ("rmsnorm_desc", NB, buf(512, 511, 128, 512, 512, 128), "dy"),
    ("rmsnorm_desc", NB, buf(512, 512, 128, 511, 512, 128), "dh"), ("rmsnorm_desc", NB, buf(512, 512, 128, 512, 511, 128), "dx"),
    ("rmsnorm_desc", NB, buf(512, 512, 128, 512, 512, 127), "dweight"),
    ("rmsnorm_desc", NB, [[1 << 24, BIG], [2 << 24, BIG], [3 << 24, BIG], [4 << 24, BIG], [5 << 24, BIG], [5 << 24, BIG]], "dweight"),
    ("muon_desc", M, buf(*[256] * 5), "expected args"), ("muon_desc", dict(M, momentum=0.0), buf(*[256] * 6), "expected args"),
    ("muon_desc", M, buf(256, 256, 256, 255, 256, 256), "smaller"), ("muon_desc", M, [[1 << 24, 256]] * 6, "twice"),
    ("muon_desc", M, [[a << 24, 256] for a in (1, 2, 3, 4, 1, 6)], "twice"), ("muon_desc", M, [[a << 24, 256] for a in (1, 2, 3, 1, 5, 6)], "gradient"),
]
ACCEPTED = [
    ("embedding_desc", E, buf(16, 320, 128)), ("embedding_desc", EB, buf(16, 128, 320)), ("rmsnorm_desc", dict(N, has_residual=True), [[1 << 24, 512], [2 << 24, 512], [2 << 24, 512], [1 << 24, 512]]),
    ("rmsnorm_desc", dict(N, quant=True, group=24), buf(512, 256, 48)), ("rmsnorm_desc", NB, [[1 << 24, 512], [2 << 24, 512], [3 << 24, 128], [4 << 24, 512], [2 << 24, 512], [6 << 24, 128]]),
    ("muon_desc", M, buf(*[256] * 6)), ("muon_desc", dict(M, momentum=0.0), buf(*[256] * 4)), ("muon_desc", dict(M, coefficients=[1.5, -0.5, 0.0]), buf(*[256] * 6)),
]


@pytest.fixture(scope="module")
def answers():
    from zyx_b200 import build
    build.build()
    out = os.path.join(ROOT, "tests", "fake", "_build")
    os.makedirs(out, exist_ok=True)
    lib = os.path.join(out, "liboperator_checks_%d.so" % os.getpid())
    objects = [os.path.join(build.OBJ, n + ".cu.o") for n in ("embedding", "rmsnorm", "muon")]
    subprocess.check_call([build.NVCC, "-shared", "-o", lib, "-std=c++17", "-Xcompiler", "-fPIC", os.path.join(ROOT, "tests", "fake", "operator_checks.cpp")] + objects +
                          ["-cudart", "static", "-gencode", "arch=compute_100a,code=sm_100a"])
    try:
        cases = [dict(make=m, kw=kw, args=None) for m, kw, _ in CREATE] + [dict(make=m, kw=kw, args=a) for m, kw, a, _ in LAUNCH] + [dict(make=m, kw=kw, args=a) for m, kw, a in ACCEPTED]
        r = subprocess.run([sys.executable, os.path.join(ROOT, "tests", "fake", "operator_checks.py"), lib], input=json.dumps(cases), capture_output=True, text=True,
                           env=dict(os.environ, CUDA_VISIBLE_DEVICES=""), timeout=300)
        assert r.returncode == 0, r.stderr[-2000:]
        return json.loads(r.stdout)
    finally:
        os.remove(lib)


@pytest.mark.parametrize("i", range(len(CREATE)), ids=lambda i: "%s-%s" % (CREATE[i][0], CREATE[i][2]))
def test_creation_refuses(answers, i):
    status, text = answers[i]
    assert status == "KernelCompilation" and CREATE[i][2] in text, (status, text)


@pytest.mark.parametrize("i", range(len(LAUNCH)), ids=lambda i: "%s-%s" % (LAUNCH[i][0], LAUNCH[i][3]))
def test_launch_refuses(answers, i):
    status, text = answers[len(CREATE) + i]
    assert status == "IncorrectKernelArg" and LAUNCH[i][3] in text, (status, text)


@pytest.mark.parametrize("i", range(len(ACCEPTED)), ids=lambda i: ACCEPTED[i][0])
def test_what_is_allowed_reaches_the_launch(answers, i):
    status, text = answers[len(CREATE) + len(LAUNCH) + i]
    assert status == "KernelLaunch", (status, text)


def test_descriptors_agree_with_the_header():
    """offsetof() and sizeof() of the three descriptors, compiled from the header, equal the ctypes mirror, and the descriptor union has
    not grown (the layout that other bindings were written against)."""
    import ctypes as C
    import tempfile
    pairs = [("zyxb_embedding_desc", L.EmbeddingDesc), ("zyxb_rmsnorm_desc", L.RmsnormDesc), ("zyxb_muon_desc", L.MuonDesc)]
    lines = ['  printf("%%zu\\n", offsetof(%s, %s));' % (c, f) for c, t in pairs for f, _ in t._fields_] + ['  printf("%%zu\\n", sizeof(%s));' % c for c, _ in pairs]
    src = "#include <stdio.h>\n#include <stddef.h>\n#include \"zyxb.h\"\nint main(void) {\n" + "\n".join(lines) + "\n  return 0;\n}\n"
    with tempfile.TemporaryDirectory() as d:
        open(os.path.join(d, "t.c"), "w").write(src)
        subprocess.check_call(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), os.path.join(d, "t.c"), "-o", os.path.join(d, "t")])
        got = [int(v) for v in subprocess.check_output([os.path.join(d, "t")]).split()]
    want = [getattr(t, f).offset for _, t in pairs for f, _ in t._fields_] + [C.sizeof(t) for _, t in pairs]
    assert got == want
    assert C.sizeof(L.KernelDesc) == 8 + C.sizeof(L.GemmDesc)
