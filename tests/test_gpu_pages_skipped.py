"""A move or copy with -1 on one side is skipped, and what is out of range on the other is bad all
the same, for moves and copies alike."""
import pytest
import torch

from dense_fixtures import gen
from fronk_amd import dense
from test_gpu_kv import noise
from test_gpu_pages import by_token, ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("other", [2 ** 31 - 1, -2, -2 ** 31, 96, 2, -1])
def test_minus_one_beside_anything(other):
    cache = noise(dense.KVCache.empty(3, 2, 32, 128), 60)
    status, want = torch.zeros(1, dtype=torch.int32, device="cuda"), by_token(cache)
    there = other in (2, -1)
    for source, target in (([-1, -1], [other, -1]), ([other, -1], [-1, -1])):
        for call, bit in ((dense.kv_move, dense.BAD_SLOT), (dense.kv_copy, dense.BAD_PAGE)):
            status.zero_()
            call(cache, ints(source), ints(target), status=status)
            assert status.item() == (0 if there else bit), (call.__name__, source, target)
    for a, b in zip(by_token(cache), want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("moves", [3, 20, 64])
def test_bad_slots_beside_skipped_ones(moves):
    """One that is bad on one side and there on the other says so; all others are moved."""
    cache = noise(dense.KVCache.empty(8, 2, 32, 64), 61)
    status, parts = torch.zeros(1, dtype=torch.int32, device="cuda"), by_token(cache)
    source, target = torch.randperm(128, generator=gen(62))[:moves].tolist(), list(range(128, 128 + moves))
    source[0], target[0], source[1] = -1, 256, 256
    dense.kv_move(cache, ints(source), ints(target), status=status)
    assert status.item() == dense.BAD_SLOT
    for x in parts:
        x[128 + 2:128 + moves] = x[source[2:]]
    for a, b in zip(by_token(cache), parts):
        assert torch.equal(a, b)
