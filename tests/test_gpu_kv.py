"""The 8-bit cache on the GPU: what is written bit for bit against a search
among all codes, what is read back, and attention over it against softmax in 64
bits of the values that the cache holds."""
import pytest
import torch

from dense_fixtures import HALF, U, attend, e4m3, gen, held, near
from fronk_amd import dense

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def noise(cache, seed):
    """Fills the cache with what unwritten memory may hold: any bytes."""
    for i, t in enumerate(cache):
        t.copy_(torch.randint(0, 256, t.shape, dtype=torch.uint8, generator=gen(seed + i)))
    return cache


def places(slots, page):
    s = slots.long()
    return s // page, s % page


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("heads,page,dim,tokens", [(1, 16, 64, 1), (2, 32, 128, 37), (3, 48, 256, 65), (8, 64, 64, 5)])
def test_append_and_read(heads, page, dim, tokens, dtype):
    r = gen(1)
    pages = tokens // page + 3
    k = torch.randn(tokens, heads, dim, generator=r) * torch.exp(3 * torch.randn(tokens, heads, 1, generator=r))
    v = torch.randn(tokens, heads, dim, generator=r) * torch.exp(3 * torch.randn(tokens, heads, 1, generator=r))
    k, v = k.to(dtype), v.to(dtype)
    slots = torch.randperm(pages * page, generator=r)[:tokens].to(torch.int32)
    cache = noise(dense.KVCache.empty(pages, heads, page, dim), 2)
    before = [t.clone() for t in cache]
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    dense.kv_append(cache, k.cuda(), v.cuda(), slots.cuda(), status=status)
    torch.cuda.synchronize()
    assert status.item() == 0
    pg, at = places(slots, page)
    kc, vc, ke, ve = (t.cpu() for t in cache)
    (kv, kq, kx), (vv, vq, vx) = held(k), held(v)
    assert torch.equal(ke[pg, :, at], kx) and torch.equal(ve[pg, :, at], vx)
    zero = kq & 0x7f == 0   # a zero's sign is of no account
    assert torch.equal(kc[pg, :, at][~zero], kq[~zero]) and ((kc[pg, :, at][zero] & 0x7f) == 0).all()
    got = vc[pg, :, at // 16, :, at % 16]
    zero = vq & 0x7f == 0
    assert torch.equal(got[~zero], vq[~zero]) and ((got[zero] & 0x7f) == 0).all()
    # All other places keep their bytes.
    other = torch.ones(pages, page, dtype=torch.bool)
    other[pg, at] = False
    for now, old in ((kc, before[0].cpu()), (ke, before[2].cpu()), (ve, before[3].cpu())):
        assert torch.equal(now.transpose(1, 2)[other], old.transpose(1, 2)[other])
    flat = [x.permute(0, 2, 4, 1, 3).reshape(pages, page, heads, dim)[other] for x in (vc, before[1].cpu())]
    assert torch.equal(*flat)
    for out_type in (F32, dtype):
        rk, rv = dense.kv_read(cache, slots.cuda(), out_type)
        near(rk, kv.to(out_type), 0.0, "k")   # NaN where fp16 made an infinity of an input
        near(rv, vv.to(out_type), 0.0, "v")


@pytest.mark.parametrize("dim,heads,tokens", [(64, 3, 130), (64, 64, 130), (128, 32, 131), (256, 16, 129)])
@pytest.mark.parametrize("first", [0, 1, 4, 14, 16, 33])
def test_runs_of_slots(first, dim, heads, tokens):
    """Streams that begin at any place of a page, with a hole, a slot out of
    order and pages in any order, written and read as whole blocks, in fours or
    singly: the bytes of a search among all codes, and no others."""
    r = gen(6)
    page, pages = 48, 6
    k, v = torch.randn(tokens, heads, dim, generator=r), torch.randn(tokens, heads, dim, generator=r)
    order = torch.tensor([4, 1, 5, 0])
    place = torch.arange(tokens) + first
    slots = order[place // page] * page + place % page
    slots[60], slots[[82, 83]] = -1, slots[[83, 82]]
    cache = noise(dense.KVCache.empty(pages, heads, page, dim), 7)
    want_k, want_v = (t.cpu().clone() for t in cache[:2])
    dense.kv_append(cache, k.cuda(), v.cuda(), slots.to(torch.int32).cuda())
    live = slots >= 0
    pg, at = slots[live] // page, slots[live] % page
    (kv, kq, _), (vv, vq, _) = held(k[live]), held(v[live])
    want_k[pg, :, at], want_v[pg, :, at // 16, :, at % 16] = kq, vq
    assert torch.equal(cache[0].cpu() & 0x7f, want_k & 0x7f) and torch.equal(cache[1].cpu() & 0x7f, want_v & 0x7f)
    rk, rv = dense.kv_read(cache, slots.to(torch.int32).cuda(), F32)
    near(rk[live], kv.float(), 0.0, "k")
    near(rv[live], vv.float(), 0.0, "v")
    assert (rk[~live] == 0).all() and (rv[~live] == 0).all()


def test_append_extremes():
    """Zeros, subnormals, the largest, ties between codes, borders of the
    exponent, infinities and NaN."""
    rows = [torch.zeros(64), torch.full((64,), 2.0 ** -149), torch.full((64,), 3.4028234663852886e38),
            torch.linspace(-448, 448, 64), torch.linspace(-449, 449, 64), torch.arange(64.0) / 64 * 2.0 ** -120,
            448 * 2.0 ** -10 * torch.ones(64), torch.tensor([448.0] + [17.0 + i for i in range(63)]),
            torch.tensor([1.75] + [2.0 ** -i for i in range(63)]),
            torch.tensor([1.7500001] + [-2.0 ** -i for i in range(63)]),
            torch.tensor([1.0] * 63 + [float("inf")]), torch.tensor([float("nan")] + [1.0] * 63),
            torch.tensor([-float("inf"), float("nan")] + [1.0] * 62), -torch.arange(64.0) * 1.0625]
    x = torch.stack(rows)[:, None]
    n = len(rows)
    cache = noise(dense.KVCache.empty(1, 1, 16, 64), 3)
    slots = torch.arange(n, dtype=torch.int32).cuda()
    dense.kv_append(cache, x.cuda(), x.flip(2).cuda(), slots)
    value, code, exp = held(x)
    rk, rv = dense.kv_read(cache, slots, F32)
    assert torch.equal(cache.k_exp.cpu()[0, 0, :n], exp[:, 0]) and torch.equal(cache.v_exp.cpu()[0, 0, :n], exp[:, 0])
    # Read as fp32, which has no 2^128: the code nearest to the largest fp32.
    near(rk, value.float(), 0.0, "k")
    near(rv, value.flip(2).float(), 0.0, "v")


def test_slots_out_of_range_touch_nothing():
    cache = noise(dense.KVCache.empty(2, 1, 16, 64), 4)
    before = [t.clone() for t in cache]
    k = torch.ones(5, 1, 64, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    slots = torch.tensor([-1, 32, -2, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32).cuda()
    dense.kv_append(cache, k[:1], k[:1], slots[:1], status=status)
    assert status.item() == 0
    dense.kv_append(cache, k, k, slots, status=status)
    assert status.item() == dense.BAD_SLOT
    assert all(torch.equal(a, b) for a, b in zip(cache, before))
    status.zero_()
    rk, rv = dense.kv_read(cache, slots, F32, status=status)
    assert status.item() == dense.BAD_SLOT and (rk == 0).all() and (rv == 0).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_append_views(dtype):
    row = torch.randn(9, 2 * 128 + 5, generator=gen(5)).to(dtype).cuda()
    k, v = row[:, 1:129].unflatten(1, (2, 64)), row[:, 130:258].unflatten(1, (2, 64))
    a, b = dense.KVCache.empty(1, 2, 16, 64), dense.KVCache.empty(1, 2, 16, 64)
    slots = torch.arange(9, dtype=torch.int32).cuda()
    for c, x, y in ((a, k, v), (b, k.contiguous(), v.contiguous())):
        for t in c:
            t.zero_()
        dense.kv_append(c, x, y, slots)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


# ------------------------------------------------------------------- attend

def filled(seed, lens, kv_heads, page, dim, spread=1.0):
    """A cache with the sequences' pages scattered, the rest of it any bytes;
    and the values it holds, in 64 bits."""
    r = gen(seed)
    per = max(1, (max(lens) + page - 1) // page) + 1
    pages = len(lens) * per + 2
    cache = noise(dense.KVCache.empty(pages, kv_heads, page, dim), seed + 1)
    table = torch.randperm(pages, generator=r)[:len(lens) * per].view(len(lens), per).to(torch.int32)
    ks, vs = [], []
    for i, n in enumerate(lens):
        k = spread * torch.randn(n, kv_heads, dim, generator=r)
        v = torch.randn(n, kv_heads, dim, generator=r) * torch.exp(torch.randn(n, 1, 1, generator=r))
        at = torch.arange(n)
        slots = (table[i].long()[at // page] * page + at % page).to(torch.int32).cuda()
        dense.kv_append(cache, k.cuda(), v.cuda(), slots)
        ks.append(held(k)[0]), vs.append(held(v)[0])
    return cache, table.cuda(), ks, vs


def tolerance(want, dtype, vs, scores):
    """One rounding of the output; softmax weights that are off by the fp32
    error of a score (`scores` in magnitude, 16 roundings of its sums), of exp2
    and of sums over the tokens (64 roundings), and, for 16-bit outputs, by P's
    two bf16 parts (2^-17): relative to the largest value that is weighed."""
    top = max([float(v.abs().max()) for v in vs if v.numel()] + [0.0])
    weight = (16 * scores + 64) * U + (0 if dtype == F32 else 2.0 ** -17)
    return HALF[dtype] * want.abs() + weight * top


def compare(seed, lens, burst, heads, kv_heads, page, dim, dtype, scale=None, spread=1.0, **kw):
    cache, table, ks, vs = filled(seed, lens, kv_heads, page, dim, spread)
    q = torch.randn(len(lens) * burst, heads, dim, generator=gen(seed + 7)).to(dtype)
    scale = dim ** -0.5 if scale is None else scale
    want = attend(q, ks, vs, lens, burst, scale)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    o = dense.kv_attend(cache, q.cuda(), table, torch.tensor(lens, dtype=torch.int32).cuda(), scale=scale,
                        status=status, **kw)
    torch.cuda.synchronize()
    assert status.item() == 0
    scores = scale * float(q.double().abs().max()) * spread * 4 * dim
    near(o, want, tolerance(want, dtype, vs, scores), "o")
    return o


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 63, 64, 65, 255, 256, 257, 700])
def test_contexts(n, dtype):
    compare(10, [n], 1, 4, 2, 32, 64, dtype)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("heads,kv_heads,page,dim", [(1, 1, 16, 64), (16, 2, 64, 256), (6, 2, 48, 128), (7, 1, 16, 128),
                                                     (12, 4, 128, 64), (34, 2, 32, 64), (64, 1, 16, 256)])
def test_heads_and_pages(heads, kv_heads, page, dim, dtype):
    compare(11, [300, 45], 1, heads, kv_heads, page, dim, dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("burst", [1, 2, 3, 5, 8])
def test_bursts_over_ragged_contexts(burst, dtype):
    """Contexts shorter than the burst among them: the rows that see nothing
    are zeros."""
    o = compare(12, [8, 1, 0, 130, 3, 64, 513], burst, 8, 2, 16, 64, dtype)
    for i, n in enumerate([8, 1, 0]):
        empty = max(0, burst - n)
        assert (o[i * burst:i * burst + empty] == 0).all()


@pytest.mark.parametrize("dtype,dim", [(BF16, 256), (F32, 128), (F16, 64)])
def test_long(dtype, dim):
    compare(13, [5000], 2, 8, 1, 64, dim, dtype)


def test_max_context_bounds_the_work():
    a = compare(14, [100, 400], 2, 8, 2, 16, 64, BF16, max_context=400)
    b = compare(14, [100, 400], 2, 8, 2, 16, 64, BF16)
    assert (a.float() - b.float()).abs().max() <= 2 * HALF[BF16] * a.float().abs().max()


@pytest.mark.parametrize("spread", [30.0, 1e-20])
def test_sharp_and_flat(spread):
    """Scores that pick one token, and scores that are all alike."""
    compare(15, [321], 1, 4, 1, 16, 64, F32, scale=0.5, spread=spread)


def test_non_finite_tokens_reach_only_the_rows_that_see_them():
    lens, burst = [90], 4
    cache, table, ks, vs = filled(16, lens, 1, 16, 64)
    q = torch.randn(burst, 4, 64, generator=gen(17)).cuda()
    length = torch.tensor(lens, dtype=torch.int32).cuda()
    clean = dense.kv_attend(cache, q, table, length)
    # The burst's third token (88 of 0..89) gets an infinite value, its last a NaN key.
    bad = torch.ones(2, 1, 64, device="cuda")
    k, v = dense.kv_read(cache, slots := torch.tensor([int(table[0, t // 16]) * 16 + t % 16 for t in (88, 89)],
                                                      dtype=torch.int32).cuda(), F32)
    v[0, 0, 5], k[1, 0, 9] = float("inf"), float("nan")
    dense.kv_append(cache, k, v, slots)
    o = dense.kv_attend(cache, q, table, length)
    assert torch.equal(o[:2], clean[:2]) and torch.isnan(o[2:]).all() and bad is not None


def test_bad_pages_and_lengths():
    """A page outside the cache counts as not seen; a length outside its bound
    gives zeros. Both are named."""
    lens = [70, 70, 70]
    cache, table, ks, vs = filled(18, lens, 2, 16, 64)
    q = torch.randn(3, 4, 64, generator=gen(19))
    for bad in (-1, cache.k_codes.shape[0], 2 ** 31 - 1, -2 ** 31):
        t = table.clone()
        t[1, 2] = bad
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        o = dense.kv_attend(cache, q.cuda(), t, torch.tensor(lens, dtype=torch.int32).cuda(), status=status)
        assert status.item() == dense.BAD_PAGE
        left = torch.cat([torch.arange(32), torch.arange(48, 70)])
        want = attend(q, [ks[0], ks[1][left], ks[2]], [vs[0], vs[1][left], vs[2]], [70, 54, 70], 1, 0.125)
        near(o, want, tolerance(want, F32, vs, 0.125 * 4 * 4 * 64), "o")
    for bad in (-1, 97, 2 ** 31 - 1, -2 ** 31):
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        o = dense.kv_attend(cache, q.cuda(), table, torch.tensor([70, bad, 70], dtype=torch.int32).cuda(),
                            max_context=96, status=status)
        assert status.item() == dense.BAD_LENGTH
        assert (o[1] == 0).all() and (o[0] != 0).any() and (o[2] != 0).any()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_attend_views(dtype):
    cache, table, ks, vs = filled(20, [200, 33], 2, 16, 64)
    q = torch.randn(4, 6, 64, generator=gen(21)).to(dtype)
    want = attend(q, ks, vs, [200, 33], 2, 0.125)
    wide = torch.zeros(4, 6 * 64 + 3, dtype=dtype).cuda()
    view = wide[:, 1:385].unflatten(1, (6, 64))
    view.copy_(q)
    out = torch.full((6, 4, 66), 2.0, dtype=dtype).cuda()
    length = torch.tensor([200, 33], dtype=torch.int32).cuda()
    o = dense.kv_attend(cache, view, table, length, out=out[:, :, 1:65].transpose(0, 1))
    near(o, want, tolerance(want, dtype, vs, 0.125 * 4 * 4 * 64), "o")
    assert (out[:, :, 0] == 2.0).all() and (out[:, :, 65] == 2.0).all()
    # Tables with a wider row, and one sequence of it.
    big = torch.full((2, table.shape[1] + 3), -9, dtype=torch.int32).cuda()
    big[:, :table.shape[1]] = table
    again = dense.kv_attend(cache, view, big[:, :table.shape[1]], length)
    assert torch.equal(again, o.contiguous())
    one = dense.kv_attend(cache, view[2:], big[1:, :table.shape[1]], length[1:])
    near(one, want[2:], tolerance(want[2:], dtype, vs, 0.125 * 4 * 4 * 64), "one sequence")


def test_decode_through_a_graph():
    """Append and attend captured once, replayed token by token with lengths
    and slots that change, against eager calls."""
    torch.manual_seed(22)
    cache, table, _, _ = filled(23, [60, 200], 2, 16, 128)
    copy = dense.KVCache(*(t.clone() for t in cache))
    k, v = (torch.randn(2, 2, 128, device="cuda").to(BF16) for _ in range(2))
    q = torch.randn(2, 8, 128, device="cuda").to(BF16)
    lens = torch.tensor([60, 200], dtype=torch.int32).cuda()
    slots = torch.zeros(2, dtype=torch.int32).cuda()

    def step(c):
        dense.kv_append(c, k, v, slots)
        return dense.kv_attend(c, q, table, lens)

    step(copy)
    torch.cuda.synchronize()
    copy = dense.KVCache(*(t.clone() for t in cache))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        o = step(cache)
    for n in range(4):
        lens += 1
        at = (lens - 1).long()
        slots.copy_(table[torch.arange(2, device="cuda"), at // 16] * 16 + (at % 16).int())
        k.normal_(), v.normal_(), q.normal_()
        graph.replay()
        torch.cuda.synchronize()
        want = step(copy)
        torch.cuda.synchronize()
        assert torch.equal(o, want) and torch.isfinite(o).all()
        assert all(torch.equal(a, b) for a, b in zip(cache, copy))


def test_refusals():
    cache, table, _, _ = filled(24, [20], 2, 16, 64)
    q = torch.zeros(1, 4, 64, device="cuda")
    length = torch.tensor([20], dtype=torch.int32).cuda()
    assert dense.kv_attend(cache, q[:0], table[:0], length[:0]).shape == (0, 4, 64)
    for bad in (dict(q=q[:, :3]), dict(q=q[:, :, :32]), dict(q=q.double()), dict(table=table.long()),
                dict(lengths=length.long()), dict(max_context=10 ** 6), dict(q=torch.zeros(9, 4, 64, device="cuda")),
                dict(scale=float("nan")), dict(out=q[:, :2]), dict(cache=(cache[0], cache[1], cache[2], cache[3].int())),
                dict(cache=(cache[0], cache[1][:, :, :, :32], *cache[2:]))):
        with pytest.raises(ValueError):
            dense.kv_attend(**{**dict(cache=cache, q=q, table=table, lengths=length), **bad})
    k = torch.zeros(2, 2, 64, device="cuda")
    slots = torch.zeros(2, dtype=torch.int32, device="cuda")
    for bad in (dict(k=k[:1]), dict(v=k.half()), dict(slots=slots[:1]), dict(slots=slots.long()), dict(k=k[:, :1])):
        with pytest.raises(ValueError):
            dense.kv_append(**{**dict(cache=cache, k=k, v=k, slots=slots), **bad})
