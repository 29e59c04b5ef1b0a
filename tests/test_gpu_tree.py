"""Attention of trees of drafts over the cache against softmax in 64 bits of the
values that it holds: types, head sizes and groups, trees of one to 64, pages that
end inside a tile, stretches, rows that see nothing, unseen garbage, bad lengths,
pages and offsets, and graphs."""
import random

import pytest
import torch

from attention_fixtures import attend_tolerance, random_tree, tree, words
from dense_fixtures import HALF, gen, near
from fronk_amd import dense
from test_gpu_kv import noise

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
WEIGHTS = {F32: 2.0 ** -23, F16: 2.0 ** -16, BF16: HALF[BF16]}   # three, two and one bf16 parts


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def starts(lens):
    return ints([sum(lens[:i]) for i in range(len(lens) + 1)])


def filled(seed, lengths, kv_heads, page, dim, spread=2.0):
    """(cache, table, k, v): sequences of these lengths in pages in any order among noise,
    and the values that are held, per sequence."""
    r = gen(seed)
    per = max(1, (max(lengths) + page - 1) // page)
    cache = noise(dense.KVCache.empty(len(lengths) * per + 2, kv_heads, page, dim), seed)
    table = torch.randperm(len(lengths) * per + 2, generator=r)[:len(lengths) * per].view(-1, per).to(torch.int32)
    k, v = [], []
    for row, n in zip(table, lengths):
        at = torch.arange(n)
        slots = (row[at // page] * page + at % page).to(torch.int32).cuda()
        x, y = (torch.randn(n, kv_heads, dim, generator=r) * torch.exp(spread * torch.randn(n, kv_heads, 1, generator=r)) for _ in range(2))
        x /= x.norm(dim=-1, keepdim=True).clamp(min=1e-3) / dim ** 0.5
        dense.kv_append(cache, x.cuda(), y.cuda(), slots)
        x, y = dense.kv_read(cache, slots, F32)
        k.append(x.cpu()), v.append(y.cpu())
    return cache, table.cuda(), k, v


def check(got, q, k, v, masks, lens, scale, what="o"):
    o, size, terms = tree(q, k, v, masks, lens, scale)
    near(got, o, attend_tolerance(o, size, terms, BF16 if q.dtype == F16 else q.dtype, WEIGHTS[q.dtype], q.shape[2],
                                  max(x.shape[0] for x in k), 0.0) + (HALF[F16] - HALF[BF16] if q.dtype == F16 else 0) * o.abs(), what)


def trees(seed, lens):
    r = random.Random(seed)
    return [m for n in lens for m in random_tree(r, n)]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(6, 2, 64, 16), (5, 1, 128, 48), (4, 2, 256, 64), (8, 1, 256, 32), (64, 1, 64, 128)])
def test_trees(heads, kv_heads, dim, page, dtype):
    """Of unequal sizes behind unequal contexts, none before some."""
    lens, before = [1, 5, 64, 33, 2, 0, 16], [100, 0, 37, 300, 15, 9, 64]
    lengths = [a + b for a, b in zip(lens, before)]
    cache, table, k, v = filled(1, lengths, kv_heads, page, dim)
    masks = trees(2, lens)
    q = torch.randn(sum(lens), heads, dim, generator=gen(3)).to(dtype)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = dense.kv_attend_tree(cache, q.cuda(), words(masks).cuda(), table, ints(lengths), offsets=starts(lens), scale=0.2, status=status)
    assert status.item() == 0 and got.dtype == dtype
    check(got, q, k, v, masks, lens, 0.2)


@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F16, 256), (F32, 64), (F32, 256)])
@pytest.mark.parametrize("drafts,length", [(1, 1), (3, 3000), (64, 64), (20, 2065), (8, 700)])
def test_one_stream(dtype, dim, drafts, length):
    """Without offsets; long contexts go in stretches."""
    cache, table, k, v = filled(4, [length], 2, 64, dim)
    masks = trees(5, [drafts])
    q = torch.randn(drafts, 8, dim, generator=gen(6)).to(dtype)
    got = dense.kv_attend_tree(cache, q.cuda(), words(masks).cuda(), table, ints([length]))
    check(got, q, k, v, masks, [drafts], dim ** -0.5)


def test_a_chain_is_a_burst():
    """A tree of one branch sees what a burst's tokens see."""
    lengths = [77, 500, 8]
    cache, table, k, v = filled(7, lengths, 2, 32, 128)
    q = torch.randn(3 * 8, 4, 128, generator=gen(8)).to(BF16)
    chain = words([(1 << b + 1) - 1 for b in range(8)] * 3).cuda()
    a = dense.kv_attend_tree(cache, q.cuda(), chain, table, ints(lengths), max_tokens=8)
    check(a, q, k, v, chain.tolist(), [8] * 3, 128 ** -0.5)
    b = dense.kv_attend(cache, q.cuda(), table, ints(lengths))
    check(b, q, k, v, chain.tolist(), [8] * 3, 128 ** -0.5)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("scale", [0.0, -0.5, 4.0])
def test_scales(dtype, scale):
    cache, table, k, v = filled(9, [90], 1, 16, 64)
    masks = trees(10, [7])
    q = torch.randn(7, 2, 64, generator=gen(11)).to(dtype)
    got = dense.kv_attend_tree(cache, q.cuda(), words(masks).cuda(), table, ints([90]), scale=scale)
    check(got, q, k, v, masks, [7], scale)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_words_that_hide(dtype):
    """A draft that sees only others, none at all, or itself alone; bits behind the drafts; and drafts that
    none sees, whose places hold anything."""
    lens, before = [6, 6], [40, 0]
    cache, table, k, v = filled(12, [46, 6], 1, 16, 64)
    masks = [0, 1, ~0b111 & (1 << 64) - 1, 0b11, 1 << 63, 0b100100] + [0, 0b10, 1 << 40, 0b1, 0b110000, 0]
    # Draft 3 of the first and 2, 3 of the second are seen by none of those below.
    masks[2] = ~0b1111 & (1 << 64) - 1
    for i, j in ((0, 43), (1, 2), (1, 3)):
        page, at = int(table[i, j // 16]), j % 16
        for t, shape in zip(cache, ((0, slice(None), at), (0, slice(None), at // 16, slice(None), at % 16), (0, slice(None), at), (0, slice(None), at))):
            t[(page,) + shape[1:]] = 255
        k[i][j], v[i][j] = 0.0, 0.0
    q = torch.randn(12, 3, 64, generator=gen(13)).to(dtype)
    got = dense.kv_attend_tree(cache, q.cuda(), words(masks).cuda(), table, ints([46, 6]), max_tokens=6)
    check(got, q, k, v, masks, lens, 0.125)
    assert (got[[6, 8, 11]] == 0).all()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_values_that_are_not_finite(dtype):
    """A draft held with infinity or NaN, in k or v, reaches the drafts that see it; a token before them all."""
    lens, lengths = [9, 9], [60, 41]
    masks = trees(14, lens)
    q = torch.randn(18, 2, 128, generator=gen(15)).to(dtype)
    for where in "kv":
        cache, table, k, v = filled(16, lengths, 1, 16, 128)
        clean = dense.kv_attend_tree(cache, q.cuda(), words(masks).cuda(), table, ints(lengths), max_tokens=9).cpu()
        bad = torch.randn(1, 1, 128, generator=gen(17))
        bad[0, 0, 3] = float("inf")
        fine = torch.randn(1, 1, 128, generator=gen(18))
        j = 55   # draft 4 of the first
        slot = ints([int(table[0, j // 16]) * 16 + j % 16])
        held = [x[0][j:j + 1].cuda() for x in (k, v)]
        dense.kv_append(cache, bad.cuda() if where == "k" else held[0], bad.cuda() if where == "v" else held[1], slot)
        got = dense.kv_attend_tree(cache, q.cuda(), words(masks).cuda(), table, ints(lengths), max_tokens=9).cpu()
        hit = torch.tensor([i < 9 and bool(masks[i] >> 4 & 1) for i in range(18)])
        assert hit.any() and torch.isnan(got[hit]).all() and torch.equal(got[~hit], clean[~hit]), where
        slot = ints([int(table[1, 0]) * 16 + 5])
        dense.kv_append(cache, fine.cuda() if where == "v" else bad.cuda(), fine.cuda() if where == "k" else bad.cuda(), slot)
        got = dense.kv_attend_tree(cache, q.cuda(), words(masks).cuda(), table, ints(lengths), max_tokens=9).cpu()
        assert torch.isnan(got[9:]).all()


def test_bad_lengths_pages_and_offsets():
    lens, lengths = [4, 4, 4], [40, 50, 30]
    cache, table, k, v = filled(19, lengths, 2, 16, 64)
    masks = trees(20, lens)
    q = torch.randn(12, 4, 64, generator=gen(21)).to(BF16)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")

    def run(lengths=lengths, table=table, **kw):
        out = torch.full((12, 4, 64), 9.0, dtype=BF16, device="cuda")
        status.zero_()
        dense.kv_attend_tree(cache, q.cuda(), words(masks).cuda(), table, ints(lengths), out=out, status=status, **kw)
        return out.cpu(), status.item()

    want, bad = run(offsets=starts(lens))
    assert bad == 0
    check(want, q, k, v, masks, lens, 0.125)
    for n in (3, 0, -1, 65, 2 ** 31 - 1, -2 ** 31):
        got, bad = run([40, n, 30])
        assert bad == dense.BAD_LENGTH and (got[4:8] == 0).all() and torch.equal(got[:4], want[:4]) and torch.equal(got[8:], want[8:])
    got, bad = run(max_context=40)
    assert bad == dense.BAD_LENGTH and (got[4:8] == 0).all() and torch.equal(got[:4], want[:4])
    for offsets, kept in (([0, 4, 3, 12], (0, 4)), ([0, 4, 8, 13], (0, 8)), ([-1, 4, 8, 12], (4, 12)), ([0, 4, 8, -5], (0, 8)), ([4, 0, 8, 12], (8, 12))):
        got, bad = run(offsets=ints(offsets), max_tokens=4)
        a, b = kept
        if offsets[0] == 4:
            assert bad == dense.BAD_OFFSET and (got[:8] == 9).all()
            continue
        assert bad == dense.BAD_OFFSET and torch.equal(got[a:b], want[a:b]) and (got[:a] == 9).all() and (got[b:] == 9).all(), offsets
    got, bad = run(offsets=starts([4, 4, 4]), max_tokens=3)
    assert bad == dense.BAD_OFFSET and (got == 9).all()
    # A page outside the cache is not seen.
    for page in (-1, cache.k_codes.shape[0], 2 ** 31 - 1, -2 ** 31):
        other = table.clone()
        other[1, 1] = page
        got, bad = run(table=other)
        assert bad == dense.BAD_PAGE
        x, y = [k[0], torch.cat([k[1][:16], k[1][32:]]), k[2]], [v[0], torch.cat([v[1][:16], v[1][32:]]), v[2]]
        check(got, q, x, y, masks, lens, 0.125)


@pytest.mark.parametrize("sequences,longest", [(2, 3000), (70, 1400), (70, 200), (200, 700), (520, 300)])
def test_ragged_batches(sequences, longest):
    """One long context among short ones, sequences without drafts, and an offset out of order behind
    the first 64: rows of the others and behind the last stay as they are."""
    r = random.Random(sequences)
    lens = [r.choice((0, 1, 1, 2, 5, 9)) for _ in range(sequences)]
    lens[1] = 17
    lengths = [n + r.randint(0, 40) for n in lens]
    lengths[1] = longest
    cache, table, k, v = filled(31, lengths, 1, 16, 64)
    masks, total = trees(32, lens), sum(lens)
    q = torch.randn(total + 3, 3, 64, generator=gen(33)).to(BF16)
    w = words(masks + [1, 1, 1]).cuda()
    out, status = torch.full((total + 3, 3, 64), 9.0, dtype=BF16, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    call = lambda offsets: dense.kv_attend_tree(cache, q.cuda(), w, table, ints(lengths), offsets=offsets, max_tokens=20, out=out, status=status)
    want = call(starts(lens)).cpu()
    assert status.item() == 0 and (want[total:] == 9).all()
    check(want[:total], q[:total], k, v, masks, lens, 0.125)
    if sequences > 66:
        offsets = starts(lens)
        offsets[66] -= 20   # ends before it, and all that begin below an earlier one
        out.fill_(9.0)
        got = call(offsets).cpu()
        at = offsets.tolist()
        bad = [max([0] + at[:s]) > at[s] or not 0 <= at[s + 1] - at[s] <= 20 for s in range(sequences)]
        assert status.item() == dense.BAD_OFFSET and bad[65] and bad[66]
        kept = torch.zeros(total + 3, dtype=torch.bool)
        for s in range(sequences):
            if not bad[s]:
                kept[at[s]:at[s + 1]] = True
        assert (got[~kept] == 9).all()
        # (which may be cut at other places)
        check(torch.where(kept[:, None, None], got, want)[:total], q[:total], k, v, masks, lens, 0.125, "kept")


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("shift", [0, 1])
def test_strides(dtype, shift):
    lens, lengths = [10, 3], [60, 33]
    cache, table, k, v = filled(22, lengths, 2, 16, 64)
    masks = trees(23, lens)
    flat = torch.randn(13 * 400 + 8, generator=gen(24)).to(dtype)
    view = lambda t: t[shift:shift + 13 * 400].view(13, 400)[:, 16:16 + 256].unflatten(1, (4, 64))
    out = torch.full((15, 5, 64 + 8), 5.0, dtype=dtype, device="cuda")
    place = out[1:14, :4, shift:shift + 64]
    wide = torch.full((2, table.shape[1] + 3), -7, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    got = dense.kv_attend_tree(cache, view(flat.cuda()), words(masks).cuda(), wide[:, :table.shape[1]], ints(lengths), offsets=starts(lens), out=place)
    check(got, view(flat), k, v, masks, lens, 0.125)
    place.fill_(5.0)
    assert (out == 5.0).all()


def test_places_past_32_bits():
    """The last pages of a cache of 5 GB a kind."""
    cache = dense.KVCache.empty(40001, 8, 64, 256)
    table = ints([[40000, 3, 39998]])
    r = gen(25)
    x, y = torch.randn(150, 8, 256, generator=r), torch.randn(150, 8, 256, generator=r)
    at = torch.arange(150)
    slots = (table[0].cpu()[at // 64] * 64 + at % 64).to(torch.int32).cuda()
    dense.kv_append(cache, x.cuda(), y.cuda(), slots)
    x, y = (t.cpu() for t in dense.kv_read(cache, slots, F32))
    masks = trees(26, [12])
    q = torch.randn(12, 16, 256, generator=r).to(BF16)
    got = dense.kv_attend_tree(cache, q.cuda(), words(masks).cuda(), table, ints([150]))
    check(got, q, [x], [y], masks, [12], 1 / 16)


def test_refusals():
    cache, table, _, _ = filled(27, [20], 2, 16, 64)
    q, w, n = torch.randn(4, 4, 64, device="cuda"), words([1, 3, 7, 15]).cuda(), ints([20])
    two, lengths = table.expand(2, 2).contiguous(), ints([20, 20])
    for args, kw in (((q, w.int(), table, n), {}), ((q, w[:3], table, n), {}), ((q[..., :32], w, table, n), {}), ((q[:, :3], w, table, n), {}),
                     ((q, w, table.long(), n), {}), ((q, w, table[0], n), {}), ((q, w, table, lengths), {}), ((q, w, table, n), dict(max_tokens=3)),
                     ((q, w, table, n), dict(offsets=starts([2, 2]))), ((q, w, table, n), dict(max_context=33)), ((q, w, table, n), dict(out=q)),
                     ((q, w, table, n), dict(offsets=starts([4]), max_tokens=65)), ((q[:3], w[:3], two, lengths), {}), ((q, w, table, n), dict(scale=float("inf"))),
                     ((q, w.cpu(), table, n), {}), ((q.expand(4, 4, 64)[:1].expand(65, 4, 64), w[:1].expand(65).contiguous(), table, n), {}),
                     ((q, w, table, n), dict(out=q.half())), ((q, w, table, n), dict(status=torch.zeros(2, dtype=torch.int32, device="cuda")))):
        with pytest.raises(ValueError):
            dense.kv_attend_tree(cache, *args, **kw)
    with pytest.raises(ValueError, match="gradient"):
        dense.kv_attend_tree(cache, q.clone().requires_grad_(), w, table, n)
    assert dense.kv_attend_tree(cache, q[:0], w[:0], table[:0], n[:0]).shape == (0, 4, 64)
    assert dense.kv_attend_tree(cache, q[:0], w[:0], table, n).shape == (0, 4, 64)
    out = torch.empty_like(q)
    before = out._version, cache.k_codes._version
    dense.kv_attend_tree(cache, q, w, table, n, out=out)
    assert out._version > before[0] and cache.k_codes._version == before[1]


def test_replays():
    """A captured call follows its tree, table and lengths; two graphs beside eager calls."""
    lens = [5, 8]
    cache, table, k, v = filled(28, [3000, 900], 2, 64, 128)
    lengths = ints([3000, 900])
    q = torch.randn(13, 8, 128, generator=gen(29)).to(BF16)
    a, w, offsets = q.cuda(), words(trees(30, lens)).cuda(), starts(lens)
    call = lambda: dense.kv_attend_tree(cache, a, w, table, lengths, offsets=offsets, max_tokens=8)
    call()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call())
        graphs.append(g)
    for step in range(3):
        masks = trees(40 + step, lens)
        w.copy_(words(masks))
        m = [3000 - 700 * step, 900 - 440 * step]
        lengths.copy_(ints(m))
        want = call()
        for g, o in zip(graphs, outs):
            o.zero_()
            g.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want)
        check(want, q, [x[:n] for x, n in zip(k, m)], [x[:n] for x, n in zip(v, m)], masks, lens, 128 ** -0.5)
