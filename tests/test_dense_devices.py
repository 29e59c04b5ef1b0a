"""The torch side of the dense operators without a GPU: fronk_amd._dense beside a
library that only notes its calls, and tensors that only say where they are."""
import os
import shutil
import subprocess
import sys

import pytest

import fronk_amd

HERE = os.path.dirname(fronk_amd.__file__)
NAMES = ["fr_hip_delta_rule", "fr_hip_q4_product", "fr_hip_kv_append", "fr_hip_kv_read", "fr_hip_kv_attend"]
STUB = "".join(f"int {n}(void) {{ ++calls; return 0; }}\n" for n in NAMES) + \
    "".join(f"unsigned long {n}(void) {{ return 0; }}\n" for n in
            ("fr_hip_delta_workspace", "fr_hip_q4_workspace", "fr_hip_kv_workspace"))
STUB = "int calls, device;\nint fr_hip_device(void) { return device; }\n" + STUB

BEGIN = """
import ctypes, sys, torch
from torch._subclasses import FakeTensorMode
sys.path.insert(0, {folder!r})
stub = ctypes.CDLL({folder!r} + "/libfronk_hip.so")
calls, device = ctypes.c_int.in_dll(stub, "calls"), ctypes.c_int.in_dll(stub, "device")
import _dense
_dense.bind(lambda d: None, lambda d: 0)


def made(gpu):
    mode = FakeTensorMode()
    with mode:
        def t(*shape, dtype=torch.bfloat16):
            return torch.empty(*shape, dtype=dtype, device=f"cuda:{{gpu}}")
        u8, i32, f32 = torch.uint8, torch.int32, torch.float32
        x, w, s = t(2, 64), t(8, 32, dtype=u8), t(8, 1, dtype=torch.float16)
        q, v, g = t(3, 2, 64), t(3, 2, 32), t(3, 2, dtype=f32)
        cache = (t(2, 1, 16, 64, dtype=u8), t(2, 1, 1, 64, 16, dtype=u8), t(2, 1, 16, dtype=u8), t(2, 1, 16, dtype=u8))
        kv, slots, table, length = t(3, 1, 64), t(3, dtype=i32), t(3, 1, dtype=i32), t(3, dtype=i32)
    def within(f):
        def call(*a):
            with mode:
                return f(*a)
        return call
    return {{
        "delta_rule": (within(_dense.delta_rule), [q, q, v, g, g, None, None, None, None, None, None, False, None, None]),
        "q4_product": (within(_dense.q4_product), [x, w, s, None, None]),
        "kv_append": (within(_dense.kv_append), [cache, kv, kv, slots, None]),
        "kv_read": (within(_dense.kv_read), [cache, slots, torch.bfloat16, None]),
        "kv_attend": (within(_dense.kv_attend), [cache, q, table, length, None, None, None, None])}}
"""


@pytest.fixture(scope="module")
def folder(tmp_path_factory):
    d = tmp_path_factory.mktemp("stub")
    (d / "stub.c").write_text(STUB)
    subprocess.run(["gcc", "-shared", "-fPIC", str(d / "stub.c"), "-o", str(d / "libfronk_hip.so")], check=True)
    # A copy of the extension, so that the library beside it is the one that it finds.
    shutil.copy(os.path.join(HERE, "_dense.so"), d / "_dense.so")
    return d


def run(folder, code):
    r = subprocess.run([sys.executable, "-c", BEGIN.format(folder=str(folder)) + code], capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    return r.stdout


def test_tensors_of_another_gpu_are_refused(folder):
    run(folder, """
for engine, gpu in ((0, 1), (1, 0)):
    device.value = engine
    for name, (f, args) in made(gpu).items():
        try:
            f(*args)
        except ValueError as e:
            assert f"tensors are on GPU {gpu}" in str(e) and f"engine on GPU {engine}" in str(e), (name, str(e))
        else:
            raise AssertionError(name + " was not refused")
assert calls.value == 0
""")


def test_an_engine_that_is_not_open_refuses_nothing(folder):
    """What opens it is the call itself."""
    run(folder, """
device.value = -2
for n, (f, args) in enumerate(made(0).values()):
    f(*args)
    assert calls.value == n + 1
""")


def test_what_autograd_would_follow_is_refused(folder):
    """Each floating-point argument of each call; under no_grad it is not."""
    run(folder, """
import torch.autograd.forward_ad as fwd
seen = 0
for name, (f, args) in made(0).items():
    for i, t in enumerate(args):
        if not torch.is_tensor(t) or not t.is_floating_point():
            continue
        seen += 1
        t.requires_grad_()
        try:
            f(*args)
        except ValueError as e:
            assert "gradient" in str(e), (name, i, str(e))
        else:
            raise AssertionError((name, i))
        with torch.no_grad():
            f(*args)
        t.requires_grad_(False)
assert (seen, calls.value) == (5 + 2 + 2 + 1, seen), (seen, calls.value)
with fwd.dual_level():
    x = fwd.make_dual(torch.zeros(2, 64), torch.ones(2, 64))
    try:
        _dense.q4_product(x, x, x, None, None)
    except ValueError as e:
        assert "gradient" in str(e), str(e)
    else:
        raise AssertionError("a tangent")
""")


def test_what_has_no_truth_value_is_no_flag(folder):
    run(folder, """
class Neither:
    def __bool__(self):
        raise RuntimeError("ambiguous")


f, args = made(0)["delta_rule"]
args[11] = Neither()
try:
    f(*args)
except RuntimeError as e:
    assert "ambiguous" in str(e), str(e)
else:
    raise AssertionError("neither true nor false")
assert calls.value == 0
args[11] = 1
f(*args)
assert calls.value == 1
""")
