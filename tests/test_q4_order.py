"""The order in which the wavefronts of 4-bit products use their two LDS buffers,
compiled for the host: no store and read of one buffer by different wavefronts
stand between the same two barriers."""
import ctypes as C
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# Every access as (kind, block, barriers before it): 0 a store, 1 a read. As in the
# kernel, reads ahead are part of a block's products.
SHIM = r'''
#include "q4_order.h"
template <bool AHEAD> static int run(uint32_t count, int* out) {
  int n = 0, epoch = 0;
  auto note = [&](int kind, uint32_t k) { out[n++] = kind, out[n++] = (int)k, out[n++] = epoch; };
  auto skip = [](uint32_t) {};
  auto store = [&](uint32_t k) { note(0, k); };
  auto read = [&](uint32_t k) { note(1, k); };
  auto barrier = [&] { ++epoch; };
  fronk::tiles_first<AHEAD>(skip, store, barrier, read);
  for (uint32_t k = 0; k < count; ++k) {
    fronk::tiles_before<AHEAD>(k, skip, barrier, read);
    if (AHEAD) read(k + 1);
    fronk::tiles_after<AHEAD>(k, store, barrier);
  }
  return n;
}
extern "C" int order(int ahead, uint32_t count, int* out) { return ahead ? run<true>(count, out) : run<false>(count, out); }
'''


@pytest.fixture(scope="module")
def shim(tmp_path_factory):
    d = tmp_path_factory.mktemp("order")
    (d / "shim.cpp").write_text(SHIM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", "-shared", "-fPIC",
                    "-I" + os.path.join(ROOT, "fronk_amd", "csrc"), str(d / "shim.cpp"), "-o", str(d / "shim.so")],
                   check=True)
    return C.CDLL(str(d / "shim.so"))


@pytest.mark.parametrize("ahead", [0, 1])
@pytest.mark.parametrize("count", [1, 2, 3, 4, 9])
def test_a_barrier_between_stores_and_reads(shim, ahead, count):
    out = (C.c_int * 200)()
    n = shim.order(ahead, count, out)
    steps = [tuple(out[i:i + 3]) for i in range(0, n, 3)]
    stores = [(k, at) for kind, k, at in steps if kind == 0]
    reads = [(k, at) for kind, k, at in steps if kind == 1]
    for k, at in reads:
        before = [(block, e) for block, e in stores if block % 2 == k % 2 and e < at]
        assert before and before[-1][0] == k, f"block {k} is not what its buffer holds"
        assert all(e != at for block, e in stores if block % 2 == k % 2), f"block {k}'s buffer is stored to as it is read"
    assert {k for k, _ in reads} >= set(range(count))
