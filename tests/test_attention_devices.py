"""The torch side of the attention layer's operators without a GPU, as
test_dense_devices.py has the other dense ones': tensors of another GPU, and those
that autograd would follow."""
import os
import shutil
import subprocess
import sys

import pytest

import fronk_amd

HERE = os.path.dirname(fronk_amd.__file__)
NAMES = ["fr_hip_rotate", "fr_hip_prompt_attend", "fr_hip_kv_attend_tree", "fr_hip_kv_move", "fr_hip_kv_copy"]
STUB = "int calls, device;\nint fr_hip_device(void) { return device; }\n" + \
    "".join(f"int {n}(void) {{ ++calls; return 0; }}\n" for n in NAMES) + \
    "".join(f"unsigned long {n}(void) {{ return 0; }}\n" for n in ("fr_hip_prompt_workspace", "fr_hip_tree_workspace"))

BEGIN = """
import ctypes, sys, torch
from torch._subclasses import FakeTensorMode
sys.path.insert(0, {folder!r})
stub = ctypes.CDLL({folder!r} + "/libfronk_hip.so")
calls, device = ctypes.c_int.in_dll(stub, "calls"), ctypes.c_int.in_dll(stub, "device")
import _attention
_attention.bind(lambda d: None, lambda d: 0)


def made(gpu):
    mode = FakeTensorMode()
    with mode:
        def t(*shape, dtype=torch.bfloat16):
            return torch.empty(*shape, dtype=dtype, device=f"cuda:{{gpu}}")
        u8, i32 = torch.uint8, torch.int32
        q, k, v = t(3, 2, 64), t(3, 1, 64), t(3, 1, 64)
        f, words = t(32, dtype=torch.float64), t(3, dtype=torch.int64)
        cache = (t(2, 1, 16, 64, dtype=u8), t(2, 1, 1, 64, 16, dtype=u8), t(2, 1, 16, dtype=u8), t(2, 1, 16, dtype=u8))
        three, table, length, other = t(3, dtype=i32), t(1, 1, dtype=i32), t(1, dtype=i32), t(3, dtype=i32)
    def within(f):
        def call(*a):
            with mode:
                return f(*a)
        return call
    return {{
        "rotary": (within(_attention.rotary), [q, k, three, f, False, 1.0, None]),
        "prompt_attend": (within(_attention.prompt_attend), [q, k, v, None, None, None, None, None, None, None]),
        "kv_attend_tree": (within(_attention.kv_attend_tree), [cache, q, words, table, length, None, None, None, None, None, None]),
        "kv_move": (within(_attention.kv_move), [cache, three, other, None]),
        "kv_copy": (within(_attention.kv_copy), [cache, three, other, None])}}
"""


@pytest.fixture(scope="module")
def folder(tmp_path_factory):
    d = tmp_path_factory.mktemp("stub")
    (d / "stub.c").write_text(STUB)
    subprocess.run(["gcc", "-shared", "-fPIC", str(d / "stub.c"), "-o", str(d / "libfronk_hip.so")], check=True)
    shutil.copy(os.path.join(HERE, "_attention.so"), d / "_attention.so")
    return d


def run(folder, code):
    r = subprocess.run([sys.executable, "-c", BEGIN.format(folder=str(folder)) + code], capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr


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
device.value = -2   # not open: the call itself opens it
for n, (f, args) in enumerate(made(0).values()):
    f(*args)
    assert calls.value == n + 1
""")


def test_tensors_of_two_gpus_are_refused(folder):
    """Each tensor argument in turn, all others on the engine's."""
    run(folder, """
here, there = made(0), made(1)
for name, (f, args) in here.items():
    for i, x in enumerate(there[name][1]):
        swapped = [list(args)]
        if isinstance(x, tuple):
            swapped = [args[:i] + [args[i][:j] + (x[j],) + args[i][j + 1:]] + args[i + 1:] for j in range(4)]
        elif torch.is_tensor(x):
            swapped = [args[:i] + [x] + args[i + 1:]]
        else:
            continue
        for a in swapped:
            try:
                f(*a)
            except ValueError:
                pass
            else:
                raise AssertionError((name, i))
assert calls.value == 0
""")


def test_what_autograd_would_follow_is_refused(folder):
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
assert (seen, calls.value) == (3 + 3 + 1, seen), (seen, calls.value)
with fwd.dual_level():
    x = fwd.make_dual(torch.zeros(2, 1, 64), torch.ones(2, 1, 64))
    try:
        _attention.prompt_attend(x, x, x, *[None] * 7)
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


f, args = made(0)["rotary"]
args[4] = Neither()
try:
    f(*args)
except RuntimeError as e:
    assert "ambiguous" in str(e), str(e)
else:
    raise AssertionError("neither true nor false")
assert calls.value == 0
""")
