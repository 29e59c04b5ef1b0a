"""The operators of served streams one after the other, as a program has them: prompts
with rotary positions into the cache, a second chunk of them, trees of drafts, the accepted
paths moved into place, a token more, and a stream forked; each step against 64 bits of what
the cache holds. And the steps of a tree captured, beside eager ones."""
import random

import pytest
import torch

import test_gpu_prompt
import test_gpu_tree
from attention_fixtures import random_tree, words
from dense_fixtures import gen, near
from fronk_amd import dense
from test_gpu_kv import noise
from test_gpu_rotary import turned

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Streams:
    """Sequences of a cache, their lengths known to the host."""

    def __init__(self, seed, count, heads, kv_heads, dim, page, pages, dtype):
        self.gen, self.heads, self.kv_heads, self.dim, self.page, self.dtype = gen(seed), heads, kv_heads, dim, page, dtype
        self.cache = noise(dense.KVCache.empty(count * pages + 2, kv_heads, page, dim), seed)
        self.table = torch.randperm(count * pages + 2, generator=self.gen)[:count * pages].view(count, pages).to(torch.int32)
        self.lengths = [0] * count
        self.frequencies, self.magnitude = dense.rotary_frequencies(dim // 2, 10000.0, factor=4.0, context=64)

    def slots(self, i, places):
        return [int(self.table[i, p // self.page]) * self.page + p % self.page for p in places]

    def project(self, positions):
        """(q, k, v) of new tokens, with their positions; q and k checked."""
        q, k, v = (torch.randn(len(positions), h, self.dim, generator=self.gen).to(self.dtype) for h in (self.heads, self.kv_heads, self.kv_heads))
        a, b = dense.rotary(q.cuda(), k.cuda(), ints(positions), self.frequencies, magnitude=self.magnitude)
        for x, y in ((a, q), (b, k)):
            near(x, *turned(y, torch.tensor(positions), self.frequencies.cpu(), False, self.magnitude), "rotary")
        return a, b, v.cuda()

    def held(self, i, places, dtype=F32):
        return dense.kv_read(self.cache, ints(self.slots(i, places)), dtype)

    def append(self, i, k, v, places):
        dense.kv_append(self.cache, k, v, ints(self.slots(i, places)))


@pytest.mark.parametrize("other_stream", [False, True])
@pytest.mark.parametrize("heads,kv_heads,dim,page,dtype", [(6, 2, 64, 16, BF16), (8, 1, 128, 32, F16), (4, 2, 256, 64, BF16), (3, 3, 64, 16, F32)])
def test_streams(heads, kv_heads, dim, page, dtype, other_stream):
    side = torch.cuda.Stream() if other_stream else torch.cuda.current_stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run_streams(heads, kv_heads, dim, page, dtype)
    torch.cuda.current_stream().wait_stream(side)


def run_streams(heads, kv_heads, dim, page, dtype):
    s = Streams(1, 2, heads, kv_heads, dim, page, 160 // page + 2, dtype)
    scale = dim ** -0.5
    # Prompts.
    lens = [45, 70]
    q, k, v = s.project([p for n in lens for p in range(n)])
    offsets = test_gpu_tree.starts(lens)
    o = dense.prompt_attend(q, k, v, offsets=offsets, max_tokens=70)
    test_gpu_prompt.check(o, q.cpu(), k.cpu(), v.cpu(), lens, lens, scale, "prompts")
    for i, at in enumerate((0, 45)):
        s.append(i, k[at:at + lens[i]], v[at:at + lens[i]], range(lens[i]))
    # Another chunk of each, over what is held.
    more = [20, 3]
    q, k, v = s.project([lens[i] + p for i, n in enumerate(more) for p in range(n)])
    for i, at in enumerate((0, 20)):
        s.append(i, k[at:at + more[i]], v[at:at + more[i]], range(lens[i], lens[i] + more[i]))
    s.lengths = [a + b for a, b in zip(lens, more)]
    held = [s.held(i, range(n), dtype) for i, n in enumerate(s.lengths)]
    k, v = (torch.cat([x[j] for x in held]) for j in range(2))
    o = dense.prompt_attend(q, k, v, offsets=test_gpu_tree.starts(more), k_offsets=test_gpu_tree.starts(s.lengths))
    test_gpu_prompt.check(o, q.cpu(), k.cpu(), v.cpu(), more, s.lengths, scale, "chunks")
    # Trees of drafts, at their depths' positions.
    r, drafts = random.Random(2), [11, 6]
    trees = [random_tree(r, n) for n in drafts]
    q, k, v = s.project([s.lengths[i] + bin(m).count("1") - 1
                         for i, t in enumerate(trees) for m in t])
    for i, at in enumerate((0, 11)):
        s.append(i, k[at:at + drafts[i]], v[at:at + drafts[i]], range(s.lengths[i], s.lengths[i] + drafts[i]))
    there = [a + b for a, b in zip(s.lengths, drafts)]
    flat = [m for t in trees for m in t]
    o = dense.kv_attend_tree(s.cache, q, words(flat).cuda(), s.table.cuda(), ints(there), offsets=test_gpu_tree.starts(drafts))
    held = [s.held(i, range(n)) for i, n in enumerate(there)]
    test_gpu_tree.check(o, q.cpu(), [x.cpu() for x, _ in held], [y.cpu() for _, y in held], flat, drafts, scale, "drafts")
    # The deepest path of each is accepted: its tokens follow those before.
    source, target, kept = [], [], []
    for i, t in enumerate(trees):
        deepest = max(t, key=lambda m: bin(m).count("1"))
        path = [j for j in range(drafts[i]) if deepest >> j & 1]
        source.append(s.slots(i, [s.lengths[i] + j for j in path]) + [-1] * (11 - len(path)))
        target.append(s.slots(i, range(s.lengths[i], s.lengths[i] + len(path))) + [-1] * (11 - len(path)))
        at = list(range(s.lengths[i])) + [s.lengths[i] + j for j in path]
        kept.append([x[at] for x in held[i]])
        s.lengths[i] += len(path)
    dense.kv_move(s.cache, ints(source), ints(target))
    for i in range(2):
        for got, want in zip(s.held(i, range(s.lengths[i])), kept[i]):
            assert torch.equal(got, want)
    # The first stream forked: whole pages shared, the last one copied.
    last = s.lengths[0] // page
    fork = s.table[0].clone()
    spare = sorted(set(range(s.cache.k_codes.shape[0])) - set(s.table.flatten().tolist()))
    fork[last] = spare[0]
    dense.kv_copy(s.cache, s.table[0, last:last + 1].cuda(), fork[last:last + 1].cuda())
    s.table, s.lengths, kept = torch.cat([s.table, fork[None]]), s.lengths + s.lengths[:1], kept + kept[:1]
    # A token more of all three.
    assert s.lengths[0] // page == last   # (its place is on the copied page)
    q, k, v = s.project(s.lengths)
    dense.kv_append(s.cache, k, v, ints([s.slots(i, [n])[0] for i, n in enumerate(s.lengths)]))
    s.lengths = [n + 1 for n in s.lengths]
    o = dense.kv_attend(s.cache, q, s.table.cuda(), ints(s.lengths))
    for i in range(3):
        new = s.held(i, [s.lengths[i] - 1])
        kept[i] = [torch.cat([a, b]) for a, b in zip(kept[i], new)]
        for got, want in zip(s.held(i, range(s.lengths[i])), kept[i]):
            assert torch.equal(got, want)
    assert not torch.equal(kept[0][0][-1], kept[2][0][-1])
    test_gpu_tree.check(o, q.cpu(), [x.cpu() for x, _ in kept], [y.cpu() for _, y in kept], [1, 1, 1], [1, 1, 1], scale, "a token more")


@pytest.mark.parametrize("before", ["noise", "tokens"])
def test_captured(before):
    """One step of drafts as a graph: the same as eager steps on a cache of its own, bit for bit, with other
    trees, lengths and accepted places at every replay; behind tokens, or behind noise, of which outputs are NaN."""
    heads, kv_heads, dim, page, drafts = 8, 2, 128, 16, 12
    caches = [noise(dense.KVCache.empty(80, kv_heads, page, dim), 3) for _ in range(2)]
    table = torch.randperm(80, generator=gen(4))[:78].view(3, 26).to(torch.int32).cuda()
    f, _ = dense.rotary_frequencies(dim)
    q, k, v = (torch.zeros(3 * drafts, h, dim, dtype=BF16, device="cuda") for h in (heads, kv_heads, kv_heads))
    positions, slots = ints([0] * 3 * drafts), ints([-1] * 3 * drafts)
    tree, lengths = words([1] * 3 * drafts).cuda(), ints([drafts] * 3)
    source, target = ints([[-1] * 4] * 3), ints([[-1] * 4] * 3)

    def step(cache):
        a, b = dense.rotary(q, k, positions, f)
        dense.kv_append(cache, b, v, slots)
        o = dense.kv_attend_tree(cache, a, tree, table, lengths, max_tokens=drafts)
        dense.kv_move(cache, source, target)
        return o, dense.prompt_attend(a, b, v, max_tokens=drafts)

    if before == "tokens":
        x, y = (torch.randn(78 * page, kv_heads, dim, generator=gen(11)).cuda() for _ in range(2))
        places = torch.cat([p * page + torch.arange(page) for p in table.flatten().cpu()]).to(torch.int32).cuda()
        for c in caches:
            dense.kv_append(c, x, y, places)
    step(caches[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(caches[0])
    length, r, g = [0, 90, 330], random.Random(5), gen(6)
    for _ in range(5):
        masks = [random_tree(r, drafts) for _ in range(3)]
        place = lambda i, p: int(table[i, p // page]) * page + p % page
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, generator=g).to(BF16))
        tree.copy_(words([m for t in masks for m in t]))
        positions.copy_(ints([length[i] + bin(m).count("1") - 1 for i in range(3) for m in masks[i]]))
        slots.copy_(ints([place(i, length[i] + j) for i in range(3) for j in range(drafts)]))
        lengths.copy_(ints([n + drafts for n in length]))
        paths = [[j for j in range(drafts) if t[-1] >> j & 1][:4] for t in masks]
        source.copy_(ints([[place(i, length[i] + j) for j in p] + [-1] * (4 - len(p)) for i, p in enumerate(paths)]))
        target.copy_(ints([[place(i, length[i] + n) for n in range(len(p))] + [-1] * (4 - len(p)) for i, p in enumerate(paths)]))
        want = step(caches[1])
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a.view(torch.int16), b.view(torch.int16))
            assert torch.isfinite(a[:drafts]).all() and (before == "noise" or torch.isfinite(a).all())
        for a, b in zip(caches[0], caches[1]):
            assert torch.equal(a, b)
        length = [n + len(p) for n, p in zip(length, paths)]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_repeated_beside_other_work(dtype):
    """The same calls on two streams at once, with workspaces of their own: the same bits every time."""
    cache, table, _, _ = test_gpu_tree.filled(7, [4000, 300, 1700], 2, 64, 128)
    masks = words(test_gpu_tree.trees(8, [20, 3, 31])).cuda()
    q = torch.randn(54, 8, 128, generator=gen(9)).to(dtype).cuda()
    x, y, z = (t.cuda() for t in test_gpu_prompt.inputs(10, 40, 3000, 8, 2, 128, dtype))
    lengths, offsets = ints([4000, 300, 1700]), test_gpu_tree.starts([20, 3, 31])
    calls = (lambda: dense.kv_attend_tree(cache, q, masks, table, lengths, offsets=offsets),
             lambda: dense.prompt_attend(x, y, z, offsets=test_gpu_tree.starts([40]), k_offsets=test_gpu_tree.starts([3000])))
    want = [c() for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(10):
        got = []
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append([c() for c in (calls if i else calls[::-1])][::1 if i else -1])
        torch.cuda.synchronize()
        for a in got:
            assert all(torch.equal(m, n) for m, n in zip(a, want))
