"""Every width of the RMS norm and its adjoint, at row counts on both sides of the rule that spreads rows, meets a kernel that covers
the row (the launchers refuse one that does not): on the CPU, through the library's own dispatch."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def program():
    from zyx_b200 import build
    build.build()
    out = os.path.join(ROOT, "tests", "fake", "_build")
    os.makedirs(out, exist_ok=True)
    path = os.path.join(out, "rms_dispatch_%d" % os.getpid())
    subprocess.check_call([build.NVCC, "-o", path, "-std=c++17", os.path.join(ROOT, "tests", "fake", "rms_dispatch.cpp"), os.path.join(build.OBJ, "rmsnorm.cu.o"),
                           "-cudart", "static", "-gencode", "arch=compute_100a,code=sm_100a"])
    yield path
    os.remove(path)


@pytest.mark.parametrize("rows", [1, 64, 394, 473, 591, 1000, 100000])
def test_every_width_has_a_kernel_that_covers_it(program, rows):
    r = subprocess.run([program, str(rows)], capture_output=True, text=True, env=dict(os.environ, CUDA_VISIBLE_DEVICES=""), timeout=300)
    assert r.returncode == 0 and r.stderr.strip() == "%d launches" % (16384 * 2 * 3), r.stderr
    assert r.stdout == "", r.stdout[:2000]
