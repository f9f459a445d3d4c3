"""The CPython entry to the calls of packed attention and the key / value cache (csrc/pycall_attn.c) passes the arguments that ctypes passes,
each in its place: both are called against a stand-in library that writes down what it is given."""
import ctypes as C
import json
import os
import subprocess
import sys

import pytest

from tensorpencil_b200 import _lib, build

NAMES = ["tpb_attention_packed", "tpb_kv_append", "tpb_kv_attention", "tpb_kv_read"]
C_TYPE = {C.c_void_p: ("void *", "%lld", "(long long)"), C.c_int: ("int", "%d", ""), C.c_int64: ("int64_t", "%lld", "(long long)"),
          C.c_float: ("float", "%.9g", "(double)"), C.c_size_t: ("size_t", "%lld", "(long long)")}
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(_lib.__file__)))

CHILD = """
import ctypes as C, importlib.machinery, importlib.util, json, sys
stub_path, ext_path, jobs = sys.argv[1], sys.argv[2], json.loads(sys.argv[3])
from tensorpencil_b200 import _lib
stub = C.CDLL(stub_path)
stub.said.restype = C.c_char_p
loader = importlib.machinery.ExtensionFileLoader("_tpbattncall", ext_path)
ext = importlib.util.module_from_spec(importlib.util.spec_from_loader("_tpbattncall", loader))
loader.exec_module(ext)
out = []
for name, args, rc in jobs:
    fn = getattr(stub, name)
    fn.restype, fn.argtypes = _lib.SIGNATURES[name]
    got = []
    for call in (getattr(ext, name), fn):
        stub.answer(rc)
        got.append([call(*args), stub.said().decode()])
    out.append(got)
print(json.dumps(out))
"""


@pytest.fixture(scope="module")
def stand_in(tmp_path_factory):
    if not os.path.exists(_lib.ATTN_CALL_PATH):
        pytest.skip("the extension is not built for this interpreter")
    d = tmp_path_factory.mktemp("stub")
    src = "#include <stdint.h>\n#include <stddef.h>\n#include <stdio.h>\nstatic char buf[2048]; static int rc;\nvoid answer(int r) { rc = r; }\nconst char *said(void) { return buf; }\n"
    for name in NAMES:
        args = [C_TYPE[t] for t in _lib.SIGNATURES[name][1]]
        src += f"int {name}(" + ", ".join(f"{t} a{i}" for i, (t, _, _) in enumerate(args)) + ") { snprintf(buf, sizeof buf, \"" + " ".join(
            [name] + [f for _, f, _ in args]) + "\", " + ", ".join(f"{cast}a{i}" for i, (_, _, cast) in enumerate(args)) + "); return rc; }\n"
    (d / "stub.c").write_text(src)
    subprocess.run(["gcc", "-shared", "-fPIC", "-o", str(d / "libtpb200.so"), str(d / "stub.c")], check=True)
    ext = d / os.path.basename(_lib.ATTN_CALL_PATH)
    assert build.build_pycall(str(ext), str(d), build.PYCALL_ATTN_SRC)
    return str(d / "libtpb200.so"), str(ext)


def distinct(name):
    """A value of its own for every argument, larger than 32 bits where the type allows it."""
    big = {C.c_void_p: 0x7f0000000000, C.c_int64: 0x500000000, C.c_size_t: 0x900000000, C.c_int: 1000}
    return [0.5 + i if t is C.c_float else big[t] + 16 * i for i, t in enumerate(_lib.SIGNATURES[name][1])]


def test_every_argument_arrives_in_its_place(stand_in):
    jobs = [[n, distinct(n), rc] for n in NAMES for rc in (0, -3)]
    jobs += [[n, [None if t is C.c_void_p else v for t, v in zip(_lib.SIGNATURES[n][1], distinct(n))], 0] for n in NAMES]
    r = subprocess.run([sys.executable, "-c", CHILD, *stand_in, json.dumps(jobs)], check=True, capture_output=True, text=True,
                       env=dict(os.environ, PYTHONPATH=ROOT))
    for (name, args, rc), (ext, ct) in zip(jobs, json.loads(r.stdout.splitlines()[-1])):
        want = " ".join([name] + ["%.9g" % v if isinstance(v, float) else str(v or 0) for v in args])
        assert ext == ct == [rc, want]


@pytest.mark.parametrize("name", NAMES)
def test_wrong_arguments_raise_and_a_null_handle_is_refused(name):
    calls = _lib.load_attn_calls()
    fn, good = getattr(calls, name), [None, None] + [0.5 if t is C.c_float else 0 for t in _lib.SIGNATURES[name][1][2:]]
    assert fn(*good) == getattr(_lib.load(), name)(*good) == _lib.TPB_ERR_INVALID_ARG
    with pytest.raises(TypeError):
        fn(None)
    for i in range(len(good)):
        bad = list(good)
        bad[i] = "x"
        with pytest.raises((TypeError, C.ArgumentError)):
            fn(*bad)


def test_calls_go_through_ctypes_where_the_extension_is_not_built(monkeypatch):
    monkeypatch.setattr(_lib, "ATTN_CALL_PATH", _lib.ATTN_CALL_PATH + ".absent")
    monkeypatch.setattr(_lib, "_attn_calls", None)
    assert isinstance(_lib.load_attn_calls(), _lib.CtypesCalls)
