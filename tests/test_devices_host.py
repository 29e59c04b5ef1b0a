"""What is done once for each device, compiled for the host."""
import ctypes as C
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SHIM = r'''
#include "devices.h"
static fronk::Devices done;
extern "C" int act(int device, int result, int* acts) {
  return fronk::once_a_device(&done, device, [&] { return ++*acts, result; });
}
'''


def test_each_device_has_its_own_and_failures_are_not_kept(tmp_path):
    (tmp_path / "shim.cpp").write_text(SHIM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", "-shared", "-fPIC",
                    "-I" + os.path.join(ROOT, "fronk_amd", "csrc"), str(tmp_path / "shim.cpp"), "-o",
                    str(tmp_path / "shim.so")], check=True)
    act, n = C.CDLL(str(tmp_path / "shim.so")).act, C.c_int()
    # (device, what it results in, what the call returns, acts so far)
    for device, result, returned, acts in [(0, 7, 7, 1), (0, 0, 0, 2), (0, 7, 0, 2), (1, 3, 3, 3), (1, 0, 0, 4),
                                           (0, 7, 0, 4), (1, 7, 0, 4), (63, 0, 0, 5), (63, 7, 0, 5), (64, 0, 0, 6),
                                           (64, 0, 0, 7), (-2, 5, 5, 8)]:
        assert act(device, result, C.byref(n)) == returned and n.value == acts
