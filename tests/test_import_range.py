"""Which ranges of device memory zyxb_buffer_import takes, on the CPU with stand-ins of the CUDA driver's entry point: none that it
cannot check."""
import ctypes as C
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def refusal(tmp_path_factory):
    path = str(tmp_path_factory.mktemp("import_range") / "lib.so")
    subprocess.check_call(["g++", "-shared", "-fPIC", "-std=c++17", "-I/usr/local/cuda/include", os.path.join(ROOT, "tests", "fake", "import_range.cpp"), "-o", path])
    lib = C.CDLL(path)
    lib.refusal.restype, lib.refusal.argtypes = C.c_char_p, [C.c_int, C.c_uint64, C.c_uint64]
    return lambda *a: (lib.refusal(*a) or b"").decode()


BASE = 0x10000


@pytest.mark.parametrize("at,nbytes", [(BASE, 1), (BASE, 4096), (BASE + 256, 3840), (BASE + 4095, 1)])
def test_inside(refusal, at, nbytes):
    assert refusal(1, at, nbytes) == ""


@pytest.mark.parametrize("at,nbytes", [(BASE, 4097), (BASE + 256, 3841), (BASE + 4095, 2), (BASE - 256, 16), (BASE + 4096, 1), (BASE + 256, 2 ** 64 - 1), (BASE, 2 ** 64 - BASE)])
def test_outside(refusal, at, nbytes):
    assert "exceeds the allocation" in refusal(1, at, nbytes)


def test_what_cannot_be_checked_is_refused(refusal):
    assert "cuMemGetAddressRange" in refusal(0, BASE, 1)
    assert "exceeds the allocation" in refusal(2, BASE, 1)


def test_the_library_asks(refusal):
    """zyxb_buffer_import's answer is import_refusal's, with the driver's entry point or none."""
    text = open(os.path.join(ROOT, "zyx_b200", "csrc", "context.cu")).read()
    body = text[text.index("int32_t zyxb_buffer_import("):text.index("int32_t zyxb_buffer_bytes(")]
    assert "import_refusal(D.address_range" in body and "if (D.address_range)" not in body


def test_the_interop_header_and_binding_agree():
    import re
    from zyx_b200 import _lib, build
    build.build()
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "zyxb_interop.h")).read(), flags=re.S)
    declared = sorted(set(re.findall(r"\b(zyxb_[a-z0-9_]+)\s*\(", text)))
    assert declared == sorted(_lib.INTEROP_SIGNATURES)
    lib = _lib.load()
    assert all(hasattr(lib, name) for name in declared)
