"""Attention of streams that have no pages yet."""
import pytest
import torch

from dense_fixtures import gen
from fronk_amd import dense

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("per", [0, 3])
def test_tables_without_pages(per, dtype):
    cache = dense.KVCache.empty(2, 1, 16, 64)
    q = torch.randn(6, 2, 64, generator=gen(1)).to(dtype).cuda()
    table, lengths = torch.zeros(3, per, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    o = dense.kv_attend(cache, q, table, lengths, max_context=0, out=torch.full_like(q, 5.0), status=status)
    assert (o == 0).all() and status.item() == 0
    lengths[1] = 1
    o = dense.kv_attend(cache, q, table, lengths, max_context=0, status=status)
    assert (o == 0).all() and status.item() == dense.BAD_LENGTH
