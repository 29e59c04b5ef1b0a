"""Causal attention of packed prompts against softmax in 64 bits: types, head
sizes and groups, lengths around a tile and a block of rows, keys before the
queries, fewer keys than queries, strides, few rows over many keys, values that are
not finite, bad offsets, and graphs."""
import pytest
import torch

from attention_fixtures import attend_tolerance, prompt
from dense_fixtures import HALF, gen, near
from fronk_amd import dense

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
WEIGHTS = {F32: 0.0, F16: HALF[F16], BF16: HALF[BF16]}


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def starts(lens):
    return ints([sum(lens[:i]) for i in range(len(lens) + 1)])


def inputs(seed, n, m, heads, kv_heads, dim, dtype):
    r = gen(seed)
    return tuple(torch.randn(t, h, dim, generator=r).to(dtype) for t, h in ((n, heads), (m, kv_heads), (m, kv_heads)))


def check(got, q, k, v, lens, k_lens, scale, what="o"):
    o, size, terms = prompt(q, k, v, lens, k_lens, scale)
    largest = v.abs().max().item() if v.numel() else 0.0
    near(got, o, attend_tolerance(o, size, terms, q.dtype, WEIGHTS[q.dtype], q.shape[2], max(k_lens), largest), what)


LENS = [1, 33, 0, 64, 31, 130, 2, 65, 32]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("heads,kv_heads,dim", [(6, 2, 64), (5, 1, 128), (2, 2, 256), (8, 1, 256), (3, 3, 128), (64, 1, 64)])
def test_packed(heads, kv_heads, dim, dtype):
    q, k, v = inputs(1, sum(LENS), sum(LENS), heads, kv_heads, dim, dtype)
    got = dense.prompt_attend(q.cuda(), k.cuda(), v.cuda(), offsets=starts(LENS), max_tokens=max(LENS))
    assert got.dtype == dtype
    check(got, q, k, v, LENS, LENS, dim ** -0.5)
    # The launch's bound is no part of the result, nor is what says that keys are the queries' own.
    again = dense.prompt_attend(q.cuda(), k.cuda(), v.cuda(), offsets=starts(LENS), k_offsets=starts(LENS))
    check(again, q, k, v, LENS, LENS, dim ** -0.5, "again")


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_keys_before_the_queries_and_fewer(dim, dtype):
    """Sequences that see nothing at first, or have no keys at all."""
    lens, k_lens = [5, 40, 1, 130, 70, 3, 9], [69, 40, 300, 127, 0, 1, 41]
    q, k, v = inputs(2, sum(lens), sum(k_lens), 4, 2, dim, dtype)
    got = dense.prompt_attend(q.cuda(), k.cuda(), v.cuda(), offsets=starts(lens), k_offsets=starts(k_lens), max_tokens=130,
                              max_context=300, scale=0.3)
    check(got, q, k, v, lens, k_lens, 0.3)
    assert (got[5 + 40 + 1 + 130:5 + 40 + 1 + 130 + 70] == 0).all()


@pytest.mark.parametrize("n,m", [(1, 1), (1, 5000), (16, 3001), (3, 255), (129, 4097), (0, 7)])
@pytest.mark.parametrize("heads,kv_heads,dim,dtype", [(8, 1, 128, BF16), (2, 2, 256, F16), (3, 1, 64, F32), (4, 4, 128, F32)])
def test_one_sequence(heads, kv_heads, dim, dtype, n, m):
    """Without offsets; few rows over many keys go in stretches."""
    q, k, v = inputs(3, n, m, heads, kv_heads, dim, dtype)
    got = dense.prompt_attend(q.cuda(), k.cuda(), v.cuda())
    if n:
        check(got, q, k, v, [n], [m], dim ** -0.5)
    assert got.shape == q.shape


def test_sequences_of_one_length():
    q, k, v = inputs(4, 4 * 37, 4 * 50, 4, 2, 128, BF16)
    got = dense.prompt_attend(q.cuda(), k.cuda(), v.cuda(), max_tokens=37)
    check(got, q, k, v, [37] * 4, [50] * 4, 128 ** -0.5)
    got = dense.prompt_attend(q.cuda(), k.cuda(), v.cuda(), max_tokens=37, k_offsets=starts([60, 40, 13, 87]))
    check(got, q, k, v, [37] * 4, [60, 40, 13, 87], 128 ** -0.5)


def test_many_short_sequences():
    lens = [(7 * i) % 4 for i in range(700)]
    q, k, v = inputs(5, sum(lens), sum(lens), 2, 1, 64, F16)
    got = dense.prompt_attend(q.cuda(), k.cuda(), v.cuda(), offsets=starts(lens), max_tokens=3)
    check(got, q, k, v, lens, lens, 0.125)


@pytest.mark.parametrize("scale", [0.0, -0.7, 3.0, 1e-30])
def test_scales(scale):
    q, k, v = inputs(6, 70, 70, 2, 2, 64, F32)
    check(dense.prompt_attend(q.cuda(), k.cuda(), v.cuda(), scale=scale), q, k, v, [70], [70], scale)
    q, k, v = inputs(6, 70, 70, 2, 2, 64, BF16)
    check(dense.prompt_attend(q.cuda(), k.cuda(), v.cuda(), scale=scale), q, k, v, [70], [70], scale)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_growing_scores(dtype):
    """Each key's score is above all before it, by more than weights may pass the maximum by."""
    n, dim = 200, 64
    q, k = torch.zeros(n, 1, dim), torch.zeros(n, 1, dim)
    q[:, 0, 0], k[:, 0, 0] = 1.0, torch.arange(n).float() * 3
    v = torch.randn(n, 1, dim, generator=gen(7)).to(dtype)
    q, k = q.to(dtype), k.to(dtype)
    for sign in (1, -1):
        check(dense.prompt_attend(q.cuda(), k.cuda(), v.cuda(), scale=float(sign)), q, k, v, [n], [n], float(sign))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("shift,wide", [(0, True), (8, True), (1, False), (3, False)])
def test_strides(dim, dtype, shift, wide):
    """Views of one projection's rows, with and without whole 16 bytes."""
    heads, kv_heads, lens = 4, 2, [40, 1, 70]
    n, each = sum(lens), (heads + 2 * kv_heads) * dim + (24 if wide else 5)
    flat = torch.randn(n * each + 64, generator=gen(8)).to(dtype)
    rows = flat[shift:shift + n * each].view(n, each)
    q, k, v = (rows[:, a * dim:b * dim].unflatten(1, (b - a, dim)) for a, b in ((0, 4), (4, 6), (6, 8)))
    moved = flat.cuda()[shift:shift + n * each].view(n, each)
    a, b, c = (moved[:, x * dim:y * dim].unflatten(1, (y - x, dim)) for x, y in ((0, 4), (4, 6), (6, 8)))
    out = torch.full((n + 2, heads + 1, dim + shift), 7.0, dtype=dtype, device="cuda")
    place = out[1:n + 1, :heads, shift:]
    got = dense.prompt_attend(a, b, c, offsets=starts(lens), max_tokens=70, out=place)
    assert got.data_ptr() == place.data_ptr()
    check(place, q, k, v, lens, lens, dim ** -0.5)
    out[1:n + 1, :heads, shift:] = 7.0
    assert (out == 7.0).all()
    # Heads before tokens, and one key for all tokens.
    t = q.transpose(0, 1).contiguous().cuda().transpose(0, 1)
    one = b[:1].expand(n, kv_heads, dim)
    check(dense.prompt_attend(t, one, c, offsets=starts(lens), max_tokens=70), q, k[:1].expand(n, kv_heads, dim), v, lens, lens,
          dim ** -0.5)


def test_places_past_32_bits():
    n, stride = 40000, 1 << 17
    k = torch.empty((n - 1) * stride + 256, dtype=BF16, device="cuda").as_strided((n, 2, 64), (stride, 64, 1))
    v = torch.empty((n - 1) * stride + 256, dtype=BF16, device="cuda").as_strided((n, 2, 64), (stride, 64, 1))
    q, x, y = inputs(9, 20, n, 2, 2, 64, BF16)
    k.copy_(x.cuda()), v.copy_(y.cuda())
    check(dense.prompt_attend(q.cuda(), k, v), q, x, y, [20], [n], 0.125)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("dim,n,m", [(64, 150, 150), (128, 150, 190), (256, 90, 90), (128, 4, 2000)])
@pytest.mark.parametrize("value", [float("inf"), -float("inf"), float("nan")])
def test_values_that_are_not_finite(dim, n, m, dtype, value):
    """A value reaches the queries that see its key, in its dim, and nothing else."""
    q, k, v = inputs(10, n, m, 4, 2, dim, dtype)
    clean = dense.prompt_attend(q.cuda(), k.cuda(), v.cuda()).cpu()
    at, d = m - n // 2, 5
    v[at, 1, d] = value
    v[m - 1, 0, 7] = value
    got = dense.prompt_attend(q.cuda(), k.cuda(), v.cuda()).cpu()
    first = at - (m - n)
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[first:, 2:, d] = True
    hit[n - 1, :2, 7] = True
    assert torch.equal(torch.isfinite(got), ~hit)
    assert torch.equal(got[~hit], clean[~hit])


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_keys_and_queries_that_are_not_finite(dtype):
    q, k, v = inputs(11, 100, 100, 2, 1, 64, dtype)
    clean = dense.prompt_attend(q.cuda(), k.cuda(), v.cuda()).cpu()
    k[60, 0, 3], q[10, 1, 2] = float("nan"), float("nan")
    got = dense.prompt_attend(q.cuda(), k.cuda(), v.cuda()).cpu()
    hit = torch.zeros(100, 2, dtype=torch.bool)
    hit[60:] = True
    hit[10, 1] = True
    assert torch.isnan(got[hit]).all() and torch.equal(got[~hit], clean[~hit])


def test_bad_offsets():
    """A bad sequence's outputs are left, the others' are as without it."""
    q, k, v = inputs(12, 60, 60, 2, 1, 64, BF16)
    args = [x.cuda() for x in (q, k, v)]
    status = torch.zeros(1, dtype=torch.int32, device="cuda")

    def run(offsets, k_offsets, most=30, context=60):
        out = torch.full_like(args[0], 9.0)
        status.zero_()
        dense.prompt_attend(*args, offsets=ints(offsets), k_offsets=ints(k_offsets), max_tokens=most, max_context=context,
                            out=out, status=status)
        return out.cpu(), status.item()

    want, bad = run([0, 10, 30, 60], [0, 10, 30, 60])
    assert bad == 0
    check(want, q, k, v, [10, 20, 30], [10, 20, 30], 0.125)
    for offsets, k_offsets, kept in (([0, 10, 30, 61], [0, 10, 30, 60], (0, 30)), ([0, 10, 30, 60], [0, 10, 30, 61], (0, 30)),
                                     ([0, 10, 5, 60], [0, 10, 30, 60], (0, 10)), ([-1, 10, 30, 60], [0, 10, 30, 60], (10, 60)),
                                     ([0, 10, 30, 60], [0, -10, 30, 60], (30, 60)), ([0, 10, 2 ** 31 - 1, -2 ** 31], [0, 10, 30, 60], (0, 10)),
                                     ([0, 10, 30, 60], [0, 10, 30, 20], (0, 30))):
        got, bad = run(offsets, k_offsets)
        a, b = kept
        assert bad == dense.BAD_OFFSET, offsets
        assert torch.equal(got[a:b], want[a:b]) and (got[:a] == 9).all() and (got[b:] == 9).all(), (offsets, k_offsets)
    got, bad = run([0, 10, 30, 60], [0, 10, 30, 60], most=29)       # too long
    assert bad == dense.BAD_OFFSET and torch.equal(got[:30], want[:30]) and (got[30:] == 9).all()
    got, bad = run([0, 10, 30, 60], [0, 10, 30, 60], context=29)
    assert bad == dense.BAD_OFFSET and torch.equal(got[:30], want[:30]) and (got[30:] == 9).all()
    # Rows behind the last sequence, and before the first.
    got, bad = run([10, 30], [10, 30])
    assert bad == 0 and torch.equal(got[10:30], want[10:30]) and (got[:10] == 9).all() and (got[30:] == 9).all()


def test_refusals():
    q, k, v = (x.cuda() for x in inputs(13, 12, 12, 4, 2, 64, BF16))
    for args, kw in (((q, k, v[:, :, :32]), {}), ((q, k[:, :, :32], v[:, :, :32]), {}), ((q, k.float(), v.float()), {}),
                     ((q, k, v), dict(max_tokens=5)), ((q, k[:7], v[:7]), dict(max_tokens=6)), ((q, k[:7], v[:7]), dict(offsets=starts([12]))),
                     ((q, k, v), dict(max_context=11)), ((q, k, v), dict(offsets=starts([12]).long())), ((q, k, v), dict(k_offsets=starts([6, 6]))),
                     ((q[:, :3], k, v), {}), ((q, k, v), dict(scale=float("nan"))), ((q, k, v), dict(max_tokens=-1)),
                     ((q[..., :48], k[..., :48], v[..., :48]), {}), ((q, k, v), dict(out=q)), ((q, k, v), dict(out=q[:1].expand(12, 4, 64))),
                     ((q, k, v), dict(out=torch.empty(12, 4, 64, device="cuda"))), ((q, k.cpu(), v.cpu()), {}),
                     ((q[:, :, ::2], k[:, :, ::2], v[:, :, ::2]), {}), ((q[0], k, v), {})):
        with pytest.raises(ValueError):
            dense.prompt_attend(*args, **kw)
    with pytest.raises(ValueError, match="gradient"):
        dense.prompt_attend(q.float().requires_grad_(), k.float(), v.float())


def test_replays_and_streams():
    """A captured call follows what its tensors hold, beside eager ones; with a workspace (few rows)
    and without; two graphs, and another stream than the current one's."""
    heads, dim = 8, 128
    lens = [3, 60, 5]
    q, k, v = inputs(14, 68, 3000, heads, 2, dim, BF16)
    a, b, c = q.cuda(), k.cuda(), v.cuda()
    offsets, k_offsets = starts(lens), starts([2000, 60, 940])
    call = lambda: dense.prompt_attend(a, b, c, offsets=offsets, k_offsets=k_offsets, max_tokens=60, max_context=2900)
    call()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call())
        graphs.append(g)
    for step in range(4):
        k_lens = [[2000, 60, 940], [100, 2900, 0], [64, 64, 2872], [2900, 30, 70]][step]
        k_offsets.copy_(starts(k_lens))
        a.copy_(torch.randn(a.shape, generator=gen(20 + step)).to(BF16))
        want = call()
        for g, o in zip(graphs, outs):
            o.zero_()
            g.replay()
        graphs[0].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want)
        check(want, a.cpu(), k, v, lens, k_lens, dim ** -0.5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        x = a * 2
        got = dense.prompt_attend(x, b, c, offsets=offsets, k_offsets=k_offsets, max_tokens=60, max_context=2900)
    side.synchronize()
    check(got, (a * 2).cpu(), k, v, lens, k_lens, dim ** -0.5)


@pytest.mark.parametrize("dtype,dim", [(BF16, 256), (F16, 128), (F32, 64)])
def test_the_same_bits_every_time(dtype, dim):
    q, k, v = (x.cuda() for x in inputs(15, 700, 700, 4, 1, dim, dtype))
    want = dense.prompt_attend(q, k, v)
    for _ in range(5):
        assert torch.equal(dense.prompt_attend(q, k, v), want)
    check(want, q.cpu(), k.cpu(), v.cpu(), [700], [700], dim ** -0.5)
