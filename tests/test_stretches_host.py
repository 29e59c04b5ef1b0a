"""How draft trees' contexts are cut, compiled for the host: a workgroup's part has a place in the
workspace whatever the lengths are."""
import ctypes as C
import os
import random
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SHIM = r'''
#include "bounds.h"
extern "C" uint32_t bound(uint32_t longest, float part) { return fronk::stretch_bound(longest, part); }
extern "C" uint32_t stretches(uint32_t length, uint32_t bound) { return fronk::stretches(length, bound, 0xffffffffu / bound); }
'''


@pytest.fixture(scope="module")
def shim(tmp_path_factory):
    d = tmp_path_factory.mktemp("stretches")
    (d / "shim.cpp").write_text(SHIM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", "-fsanitize=undefined",
                    "-fno-sanitize-recover", "-shared", "-fPIC", "-I" + os.path.join(ROOT, "fronk_amd", "csrc"),
                    str(d / "shim.cpp"), "-o", str(d / "shim.so")], check=True)
    L = C.CDLL(str(d / "shim.so"))
    L.bound.restype = L.stretches.restype = C.c_uint32
    L.bound.argtypes, L.stretches.argtypes = (C.c_uint32, C.c_float), (C.c_uint32, C.c_uint32)
    return L


MOST = 2 ** 31 - 1 - 2 ** 20   # tokens of a context, at most


def lengths():
    r = random.Random(1)
    yield from (0, 1, 255, 256, 257, 2 ** 24 + 1, 2 ** 30 - 63, 2 ** 30, 2 ** 30 + 1, 2 ** 30 + 64, 2 ** 30 + 65, 2 ** 30 + 192, MOST - 64, MOST)
    for _ in range(2000):
        yield min(MOST, int(2 ** r.uniform(0, 31)))
        yield r.randint(2 ** 30, MOST)


def test_one_bound_leaves_all_whole(shim):
    """There are as many places as workgroups without stretches, so the largest bound has to make none."""
    for n in lengths():
        longest = (max(n, 1) + 63) & ~63
        bound = shim.bound(longest, 1.0)
        assert bound >= longest and bound % 64 == 0, n
        assert shim.stretches(n, bound) == 1, n
        assert shim.stretches(n // 3, bound) == 1


def test_stretches_cover_a_sequence(shim):
    for n in lengths():
        longest = (max(n, 1) + 63) & ~63
        for lane in (1, 5, 8, 40, 63):
            bound = shim.bound(longest, 2.0 ** (-lane / 8))
            assert bound >= 256 and bound % 64 == 0
            assert shim.stretches(n, bound) == max(1, -(-n // bound)), (n, bound)
