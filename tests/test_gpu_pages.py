"""Tokens and pages moved within the cache, bit for bit against indexing: chains of
targets that are sources, skipped and bad ones, and all that is not theirs."""
import pytest
import torch

from dense_fixtures import gen
from fronk_amd import dense
from test_gpu_kv import noise

pytestmark = pytest.mark.gpu


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def by_token(cache):
    """The cache's four parts with slots first: [slot][head][...]."""
    kc, vc, ke, ve = (t.cpu() for t in cache)
    page = kc.shape[2]
    slots = kc.shape[0] * page
    return [kc.transpose(1, 2).reshape(slots, *kc.shape[1::2]), vc.permute(0, 2, 4, 1, 3).reshape(slots, *kc.shape[1::2]),
            ke.transpose(1, 2).reshape(slots, -1), ve.transpose(1, 2).reshape(slots, -1)]


def moved(cache, source, target):
    """by_token of the cache after the moves, all of a group at once."""
    parts = by_token(cache)
    for s, t in zip(source, target):
        pairs = [(a, b) for a, b in zip(s, t) if 0 <= a < parts[0].shape[0] and 0 <= b < parts[0].shape[0]]
        if pairs:
            a, b = (torch.tensor(x) for x in zip(*pairs))
            parts = [x.index_copy(0, b, x[a]) for x in parts]
    return parts


@pytest.mark.parametrize("heads,page,dim", [(1, 16, 64), (2, 64, 256), (3, 48, 128), (8, 16, 128)])
@pytest.mark.parametrize("groups,moves", [(1, 1), (1, 7), (1, 64), (5, 8), (33, 9)])
def test_moves(heads, page, dim, groups, moves):
    per = (2 * moves + page - 1) // page
    cache = noise(dense.KVCache.empty(groups * per + 1, heads, page, dim), 1)
    r = gen(2)
    source, target = [], []
    for g in range(groups):   # ascending places to the first ones: targets are sources of others
        place = torch.randperm(2 * moves, generator=r)[:moves].sort().values
        pages = torch.arange(groups * per, dtype=torch.long).view(groups, per).flip(1)[g]
        slot = lambda x: (pages[x // page] * page + x % page).tolist()
        source.append(slot(place)), target.append(slot(torch.arange(moves)))
        if g % 2:
            source[-1][moves // 2] = -1
        if g % 3 == 1:
            target[-1][0] = -1
    want = moved(cache, source, target)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    dense.kv_move(cache, ints(source), ints(target), status=status)
    assert status.item() == 0
    for a, b in zip(by_token(cache), want):
        assert torch.equal(a, b)


def test_turns_and_swaps():
    """A ring of slots, a slot to itself, one source for many."""
    cache = noise(dense.KVCache.empty(3, 2, 32, 128), 3)
    source = [list(range(64)), [70, 71, 70, 70] + [-1] * 60]
    target = [[(i + 1) % 64 for i in range(64)], [71, 70, 72, 90] + [-1] * 60]
    want = moved(cache, source, target)
    for _ in range(1):
        dense.kv_move(cache, ints(source), ints(target))
    for a, b in zip(by_token(cache), want):
        assert torch.equal(a, b)
    flat = moved(cache, [[5, 6]], [[5, 7]])
    dense.kv_move(cache, ints([5, 6]), ints([5, 7]))
    for a, b in zip(by_token(cache), flat):
        assert torch.equal(a, b)


def test_bad_slots():
    cache = noise(dense.KVCache.empty(2, 1, 16, 64), 4)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    for source, target, bad in (([1, 32, 3], [5, 6, 7], True), ([1, 2, 3], [5, -2, 7], True), ([-2 ** 31, 2, 2 ** 31 - 1], [5, 6, 7], True),
                                ([-1, 2, 3], [40, 6, 7], True), ([-1, -1, -1], [-1, -1, -1], False), ([1, 2, 3], [-1, -1, -1], False)):
        want = moved(cache, [source], [target])
        status.zero_()
        dense.kv_move(cache, ints([source]), ints([target]), status=status)
        assert status.item() == (dense.BAD_SLOT if bad else 0), (source, target)
        for a, b in zip(by_token(cache), want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("heads,page,dim", [(1, 16, 64), (2, 64, 256), (3, 48, 128), (1, 4096, 64)])
def test_pages(heads, page, dim):
    cache = noise(dense.KVCache.empty(9, heads, page, dim), 5)
    want = [t.clone() for t in cache]
    for s, t in ((0, 7), (0, 3), (8, 2), (4, 4)):
        for x in want:
            x[t] = x[s]
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    dense.kv_copy(cache, ints([0, 0, -1, 8, 5, 4]), ints([7, 3, 6, 2, -1, 4]), status=status)
    assert status.item() == 0
    for a, b in zip(cache, want):
        assert torch.equal(a, b)
    dense.kv_copy(cache, ints([9, 1, -2, 0]), ints([1, 9, 1, 2 ** 31 - 1]), status=status)
    assert status.item() == dense.BAD_PAGE
    for a, b in zip(cache, want):
        assert torch.equal(a, b)


def test_places_past_32_bits():
    """A cache of 5 GB a kind, its last page and its first."""
    cache = dense.KVCache.empty(40001, 8, 64, 256)
    for t in cache:
        t[40000].copy_(torch.randint(0, 256, t.shape[1:], dtype=torch.uint8, generator=gen(6)))
    dense.kv_copy(cache, ints([40000]), ints([39999]))
    for t in cache:
        assert torch.equal(t[39999], t[40000])
    last = 40000 * 64 + 63
    dense.kv_move(cache, ints([last]), ints([17]))
    assert torch.equal(cache.k_codes[0, :, 17], cache.k_codes[40000, :, 63]) and torch.equal(cache.v_exp[0, :, 17], cache.v_exp[40000, :, 63])
    assert torch.equal(cache.v_codes[0, :, 1, :, 1], cache.v_codes[40000, :, 3, :, 15])


def test_refusals_and_versions():
    cache = dense.KVCache.empty(4, 1, 16, 64)
    i = ints([1, 2])
    for source, target in ((i, ints([1])), (i.long(), i.long()), (i[:, None, None], i[:, None, None]), (i, i[None]), (i.cpu(), i.cpu()),
                           (torch.zeros(65, dtype=torch.int32, device="cuda"),) * 2, (i.expand(2, 2), i.expand(2, 2))):
        with pytest.raises(ValueError):
            dense.kv_move(cache, source, target)
    for source, target in ((i, ints([1])), (i[None], i[None]), (i.float(), i.float())):
        with pytest.raises(ValueError):
            dense.kv_copy(cache, source, target)
    for call in (lambda: dense.kv_move(cache, i, ints([5, 6])), lambda: dense.kv_copy(cache, i, ints([3, 0]))):
        before = [t._version for t in cache]
        call()
        assert all(t._version > n for t, n in zip(cache, before)) and i._version == 0
    none = ints([])
    dense.kv_move(cache, none, none), dense.kv_copy(cache, none, none), dense.kv_move(cache, none.view(0, 3), none.view(0, 3))


def test_replays():
    cache = noise(dense.KVCache.empty(8, 2, 16, 64), 7)
    source, target = ints([[3, 5, 9, -1]]), ints([[0, 1, 2, -1]])
    pages, to = ints([0]), ints([4])
    dense.kv_move(cache, source, source), dense.kv_copy(cache, pages, pages)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        dense.kv_move(cache, source, target)
        dense.kv_copy(cache, pages, to)
    for step in range(3):
        source.copy_(ints([[16 + step, 20, 30, 40 - step]]))
        to.fill_(5 + step)
        want = moved(cache, source.tolist(), target.tolist())
        want = [x.view(8, 16, *x.shape[1:]).clone() for x in want]
        for x in want:
            x[5 + step] = x[0]
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(by_token(cache), want):
            assert torch.equal(a.view(b.shape), b)
