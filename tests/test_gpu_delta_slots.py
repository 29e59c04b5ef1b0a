"""Slots of the gated delta rule where there are no pools."""
import pytest
import torch

from dense_fixtures import delta_inputs
from fronk_amd import dense

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [3, 50])
def test_slots_without_pools_only_say_what_is_skipped(n):
    """Rows of a pool that another call has, at most the largest there is."""
    q, k, v, g, beta = (x.cuda() for x in delta_inputs(600, [n] * 4, 1, 2, 64, 32, torch.bfloat16))
    want = dense.delta_rule(q, k, v, g, beta, normalize=True, max_tokens=n)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = torch.full_like(v, 3.0)
    slots = torch.tensor([700, -1, 2 ** 31 - 2, 0], dtype=torch.int32).cuda()
    dense.delta_rule(q, k, v, g, beta, normalize=True, max_tokens=n, slots=slots, out=out, status=status)
    assert status.item() == 0
    for i in (0, 2, 3):
        assert torch.equal(out[i * n:(i + 1) * n], want[i * n:(i + 1) * n])
    assert (out[n:2 * n] == 3.0).all()
    slots[0] = -2
    dense.delta_rule(q, k, v, g, beta, normalize=True, max_tokens=n, slots=slots, status=status)
    assert status.item() == dense.BAD_SLOT
