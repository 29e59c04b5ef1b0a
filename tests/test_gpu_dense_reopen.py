"""The engine closed and opened again under the dense operators, in a process of
its own: other tests keep theirs."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CODE = """
import sys
sys.path[:0] = [{root!r}, {root!r} + "/tests"]
import torch
import fronk_amd as fa
from fronk_amd import dense
from dense_fixtures import delta_inputs, q4_weights

lib = fa.lib()
# Sizes whose kernels take most LDS: chunks, tiles of 64 tokens, rows with x in LDS.
args = [x.cuda() for x in delta_inputs(1, [100], 2, 4, 128, 32, torch.float32)]
w = [t.cuda() for t in q4_weights(2, 8200, 1536, 128, True)]
x = torch.randn(130, 1536, device="cuda")


def passes():
    return dense.delta_rule(*args, normalize=True), dense.q4_product(x, *w), dense.q4_product(x[:16], *w)


assert lib.fr_hip_device() == fa.STATE
first = passes()
for _ in range(2):
    torch.cuda.synchronize()
    assert lib.fr_hip_device() == 0 and lib.fr_hip_close() == fa.OK and lib.fr_hip_device() == fa.STATE
    again = passes()
    assert all(torch.equal(a, b) for a, b in zip(first, again)) and all(torch.isfinite(a).all() for a in first)
torch.cuda.synchronize()
print("the same")
"""


def test_the_engine_opened_again():
    r = subprocess.run([sys.executable, "-c", CODE.format(root=ROOT)], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and r.stdout.strip().endswith("the same"), r.stdout + r.stderr
