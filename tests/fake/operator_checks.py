"""python operator_checks.py LIBRARY < cases.json > answers.json, run with no GPU visible.
A case: {"make": descriptor builder of zyx_b200.backend, "kw": its arguments, "args": [[address, bytes], ...] or null}."""
import ctypes as C
import json
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
sys.path.insert(0, ROOT)
assert os.environ.get("CUDA_VISIBLE_DEVICES") == ""
from zyx_b200 import _lib as L  # noqa: E402
from zyx_b200 import backend as B  # noqa: E402

lib = C.CDLL(sys.argv[1])
out = []
for case in json.load(sys.stdin):
    d = getattr(B, case["make"])(**case["kw"])
    args = case["args"] or []
    ptrs = (C.c_void_p * max(1, len(args)))(*[a for a, _ in args])
    size = (C.c_uint64 * max(1, len(args)))(*[b for _, b in args])
    text = C.create_string_buffer(400)
    st = lib.check_operator(C.byref(d), ptrs, size, -1 if case["args"] is None else len(args), text, 400)
    out.append([L.ERR_NAMES.get(st, "ok" if st == 0 else str(st)), text.value.decode()])
json.dump(out, sys.stdout)
