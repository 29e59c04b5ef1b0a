"""The gated delta rule on the GPU against its recurrence in 64 bits: lengths
from none to several chunks, head layouts, types, ragged batches over slots of
a pool, views, streams, graphs, and the entries that only the device can
refuse."""
import pytest
import torch

from dense_fixtures import delta, delta_inputs, delta_tolerance, gen, near
from fronk_amd import dense

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def call(q, k, v, g, beta, state, lens, scale, normalize, **kw):
    """(o, final states) of one call over a pool that holds the sequences in
    another order, with a row to spare that must stay as it is."""
    n = len(lens)
    slots = [(3 * i + 1) % (n + 1) if (n + 1) % 3 else (i + 1) % (n + 1) for i in range(n)]
    pool = torch.full((n + 1, *state.shape[1:]), 7.0)
    pool[slots] = state
    pool = pool.cuda()
    starts = torch.tensor([sum(lens[:i]) for i in range(n + 1)], dtype=torch.int32).cuda()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    o = dense.delta_rule(q.cuda(), k.cuda(), v.cuda(), g.cuda(), beta.cuda(), pool, pool, scale=scale, offsets=starts,
                         slots=torch.tensor(slots, dtype=torch.int32).cuda(), max_tokens=max(lens),
                         normalize=normalize, status=status, **kw)
    torch.cuda.synchronize()
    assert status.item() == 0
    spare = (set(range(n + 1)) - set(slots)).pop()
    assert (pool[spare] == 7.0).all()
    return o, pool[slots]


def compare(seed, lens, key_heads, heads, dk, dv, dtype, normalize):
    q, k, v, g, beta = delta_inputs(seed, lens, key_heads, heads, dk, dv, dtype, normalize)
    state = 0.3 * torch.randn(len(lens), heads, dk, dv, generator=gen(seed + 1))
    scale = dk ** -0.5
    want, final = delta(q, k, v, g, beta, state, lens, scale, normalize)
    o, got = call(q, k, v, g, beta, state, lens, scale, normalize)
    size = max(float(final.abs().max()), 1.0)
    # |q| <= 1 once normalized; without that it is some sqrt(dk), which scale undoes.
    near(o, want, delta_tolerance(want, dtype, dk, max(lens), size), "o")
    near(got, final, delta_tolerance(final, F32, dk, max(lens), size), "state")


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("lens", [[1], [8], [63], [64], [65], [200]])
def test_lengths(lens, dtype):
    compare(10, lens, 2, 4, 128, 64, dtype, True)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("key_heads,heads,dk,dv", [(1, 1, 64, 16), (3, 9, 64, 80), (2, 2, 128, 128), (1, 4, 128, 48),
                                                   (2, 4, 256, 96), (1, 1, 256, 32)])
def test_heads(key_heads, heads, dk, dv, dtype):
    compare(20, [5, 70], key_heads, heads, dk, dv, dtype, True)


@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_ragged(dtype, normalize):
    compare(30, [0, 64, 1, 0, 129, 2, 77, 0], 2, 4, 64, 32, dtype, normalize)


@pytest.mark.parametrize("seed", range(4))
def test_bursts(seed):
    lens = [[1, 4, 2, 3], [0, 0, 1], [7] * 9, [3]][seed]
    compare(40 + seed, lens, 2, 6, 128, 128, BF16, True)


@pytest.mark.parametrize("n", [1, 90])
def test_no_states(n):
    """From zeros, and the final state dropped: o of the same tokens."""
    q, k, v, g, beta = delta_inputs(50, [n], 1, 2, 64, 32, BF16)
    want, final = delta(q, k, v, g, beta, torch.zeros(1, 2, 64, 32), [n], 0.25, True)
    size = max(float(final.abs().max()), 1.0)
    args = [x.cuda() for x in (q, k, v, g, beta)]
    pool = torch.full((1, 2, 64, 32), float("nan")).cuda()
    o = dense.delta_rule(*args, None, pool, scale=0.25, normalize=True)
    near(o, want, delta_tolerance(want, BF16, 64, n, size), "o from zeros")
    near(pool, final, delta_tolerance(final, F32, 64, n, size), "state from zeros")
    assert torch.equal(dense.delta_rule(*args, scale=0.25, normalize=True), o)


@pytest.mark.parametrize("n", [3, 150])
def test_two_pools_and_even_sequences(n):
    """state_in is left alone; without offsets all sequences are max_tokens."""
    lens = [n] * 3
    q, k, v, g, beta = delta_inputs(60, lens, 2, 2, 64, 48, F32)
    state = torch.randn(3, 2, 64, 48, generator=gen(61))
    want, final = delta(q, k, v, g, beta, state, lens, 0.125, True)
    a, b = state.cuda(), torch.empty_like(state).cuda()
    o = dense.delta_rule(*(x.cuda() for x in (q, k, v, g, beta)), a, b, scale=0.125, normalize=True, max_tokens=n)
    size = float(final.abs().max())
    near(o, want, delta_tolerance(want, F32, 64, n, size), "o")
    near(b, final, delta_tolerance(final, F32, 64, n, size), "state")
    assert torch.equal(a.cpu(), state)


@pytest.mark.parametrize("n", [2, 100])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_views(n, dtype):
    """q, k, v of one row that is offset by an odd element, heads in reverse
    stride order for o, and decays and betas of a wider row."""
    q, k, v, g, beta = delta_inputs(70, [n], 2, 4, 64, 32, dtype)
    state = torch.randn(1, 4, 64, 32, generator=gen(71))
    want, final = delta(q, k, v, g, beta, state, [n], 0.125, True)
    row = torch.zeros(n, 1 + 2 * 128 + 128 + 6, dtype=dtype).cuda()
    vq, vk, vv = row[:, 1:129].unflatten(1, (2, 64)), row[:, 129:257].unflatten(1, (2, 64)), row[:, 257:385].unflatten(1, (4, 32))
    vq.copy_(q), vk.copy_(k), vv.copy_(v)
    gb = torch.zeros(n, 11).cuda()
    gb[:, 1:5], gb[:, 6:10] = g.cuda(), beta.cuda()
    out = torch.full((4, n, 33), 5.0, dtype=dtype).cuda()
    o = dense.delta_rule(vq, vk, vv, gb[:, 1:5], gb[:, 6:10], state.cuda(), None, scale=0.125, normalize=True,
                         out=out[:, :, :32].transpose(0, 1))
    size = max(float(final.abs().max()), 1.0)
    near(o, want, delta_tolerance(want, dtype, 64, n, size), "o")
    assert (out[:, :, 32] == 5.0).all()


@pytest.mark.parametrize("n", [4, 130])
def test_decays(n):
    """Decays from none to one that empties the state at once, and beta 0 and 1."""
    q, k, v, g, beta = delta_inputs(80, [n], 2, 4, 128, 32, F32)
    g[:, 0], g[:, 1], g[n // 2, 2], g[:, 3] = 0.0, -60.0, -float("inf"), -1e-8
    beta[:, 0], beta[:, 3], beta[::2, 2] = 1.0, 0.0, 0.0
    state = torch.randn(1, 4, 128, 32, generator=gen(81))
    want, final = delta(q, k, v, g, beta, state, [n], 0.1, True)
    o, got = call(q, k, v, g, beta, state, [n], 0.1, True)
    size = float(torch.maximum(final.abs().max(), state.abs().max().double()))
    near(o, want, delta_tolerance(want, F32, 128, n, size), "o")
    near(got, final, delta_tolerance(final, F32, 128, n, size), "state")


def test_equal_keys():
    """One key for all tokens, no decay, beta 1: each token replaces the last's
    value, and the inverse that chunks need has entries that alternate."""
    n = 192
    q, k, v, g, beta = delta_inputs(85, [n], 1, 1, 64, 16, F32)
    k[:] = k[0]
    g[:], beta[:] = 0.0, 1.0
    state = torch.randn(1, 1, 64, 16, generator=gen(86))
    want, final = delta(q, k, v, g, beta, state, [n], 0.1, True)
    o, got = call(q, k, v, g, beta, state, [n], 0.1, True)
    size = max(float(final.abs().max()), 1.0)
    near(o, want, delta_tolerance(want, F32, 64, n, size), "o")
    near(got, final, delta_tolerance(final, F32, 64, n, size), "state")


@pytest.mark.parametrize("size", [1e-12, 1e12])
@pytest.mark.parametrize("n", [3, 140])
def test_magnitudes(n, size):
    """Values and states of any magnitude: the rule is linear in them."""
    q, k, v, g, beta = delta_inputs(87, [n], 1, 2, 64, 32, F32)
    v *= size
    state = size * torch.randn(1, 2, 64, 32, generator=gen(88))
    want, final = delta(q, k, v, g, beta, state, [n], 0.1, True)
    o, got = call(q, k, v, g, beta, state, [n], 0.1, True)
    top = float(final.abs().max())
    near(o, want, delta_tolerance(want, F32, 64, n, top), "o")
    near(got, final, delta_tolerance(final, F32, 64, n, top), "state")


@pytest.mark.parametrize("n", [5, 150])
def test_token_by_token_is_the_whole(n):
    """A prompt at once, and the same tokens one call each."""
    q, k, v, g, beta = (x.cuda() for x in delta_inputs(90, [n], 1, 2, 128, 64, F32))
    state = torch.randn(1, 2, 128, 64, generator=gen(91)).cuda()
    a, b = state.clone(), state.clone()
    whole = dense.delta_rule(q, k, v, g, beta, a, a, normalize=True)
    single = torch.cat([dense.delta_rule(*(x[t:t + 1] for x in (q, k, v, g, beta)), b, b, normalize=True)
                        for t in range(n)])
    size = max(float(b.abs().max()), 1.0)
    near(whole, single.cpu(), 2 * delta_tolerance(single.cpu().double(), F32, 128, n, size), "o")
    near(a, b.cpu(), 2 * delta_tolerance(b.cpu().double(), F32, 128, n, size), "state")


@pytest.mark.parametrize("n", [3, 100])
def test_bad_entries_touch_nothing(n):
    """Sequences with a bad slot or offset are left out, and named in status;
    the others are computed."""
    lens = [n] * 4
    q, k, v, g, beta = (x.cuda() for x in delta_inputs(95, lens, 1, 2, 64, 32, BF16))
    pool = torch.randn(4, 2, 64, 32, generator=gen(96)).cuda()
    good = pool.clone()
    o = dense.delta_rule(q, k, v, g, beta, good, good, normalize=True, max_tokens=n)
    starts = [0, n, 2 * n, 3 * n, 4 * n]

    def run(slots, offsets):
        p, out = pool.clone(), torch.full_like(v, 3.0)
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        dense.delta_rule(q, k, v, g, beta, p, p, normalize=True, max_tokens=n, out=out, status=status,
                         slots=torch.tensor(slots, dtype=torch.int32).cuda(),
                         offsets=torch.tensor(offsets, dtype=torch.int32).cuda())
        return p, out, status.item()

    for slots, bits in (([0, -1, 2, 3], 0), ([0, 4, 2, 3], dense.BAD_SLOT), ([0, -2, 2, 3], dense.BAD_SLOT)):
        p, out, status = run(slots, starts)
        assert status == bits
        for i in (0, 2, 3):
            assert torch.equal(p[i], good[i]) and torch.equal(out[i * n:(i + 1) * n], o[i * n:(i + 1) * n])
        assert torch.equal(p[1], pool[1]) and (out[n:2 * n] == 3.0).all()
    # Sequence 2 too long, and sequence 3 past the last token.
    p, out, status = run([0, 1, 2, 3], [0, n, 2 * n, 4 * n, 4 * n + 1])
    assert status == dense.BAD_OFFSET
    assert torch.equal(p[:2], good[:2]) and torch.equal(p[2:], pool[2:]) and (out[2 * n:] == 3.0).all()
    # A start after its end.
    p, out, status = run([0, 1, 2, 3], [0, n, n - 1, 2 * n - 1, 2 * n - 1])
    assert status == dense.BAD_OFFSET
    assert torch.equal(p[0], good[0]) and torch.equal(p[1], pool[1])


@pytest.mark.parametrize("n", [3, 100])
def test_offsets_that_go_down(n):
    """Sequences behind an offset that goes down may not share tokens with one
    before: they are left out, each time alike."""
    q, k, v, g, beta = (x.cuda() for x in delta_inputs(97, [2 * n], 1, 2, 64, 32, BF16))
    pool = torch.randn(70, 2, 64, 32, generator=gen(98)).cuda()
    good = pool[:1].clone()
    o = dense.delta_rule(q, k, v, g, beta, good, good, normalize=True)
    # The second sequence ends below its start; the later ones begin below 2 n, the
    # last of them only after 64 others of no tokens.
    offsets = torch.tensor([0, 2 * n, 1] + [2] * 67 + [2 * n], dtype=torch.int32).cuda()
    for _ in range(3):
        p, out = pool.clone(), torch.full_like(v, 3.0)
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        dense.delta_rule(q, k, v, g, beta, p, p, normalize=True, max_tokens=2 * n, out=out, status=status,
                         offsets=offsets)
        assert status.item() == dense.BAD_OFFSET
        assert torch.equal(out, o) and torch.equal(p[0], good[0]) and torch.equal(p[1:], pool[1:])


@pytest.mark.parametrize("n", [4, 200])
def test_stream_and_graph(n):
    """On a stream of its own, and replayed from a graph with eager work in
    between; every replay gives the eager result's bits."""
    args = [x.cuda() for x in delta_inputs(99, [n], 2, 4, 128, 128, BF16)]
    first = torch.randn(1, 4, 128, 128, generator=gen(100)).cuda()
    eager = first.clone()
    want = dense.delta_rule(*args, eager, eager, normalize=True)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    pool = first.clone()
    with torch.cuda.stream(s):
        s.wait_stream(torch.cuda.default_stream())
        o = dense.delta_rule(*args, pool, pool, normalize=True)
    s.synchronize()
    assert torch.equal(o, want) and torch.equal(pool, eager)
    pool = first.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = dense.delta_rule(*args, pool, pool, normalize=True)
    for _ in range(3):
        pool.copy_(first)
        o.fill_(9.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, want) and torch.equal(pool, eager)
        again = first.clone()
        assert torch.equal(dense.delta_rule(*args, again, again, normalize=True), want)
        torch.cuda.synchronize()


def test_no_tokens():
    q, k, v, g, beta = (x.cuda() for x in delta_inputs(101, [0, 0], 1, 2, 64, 32, BF16))
    a = torch.randn(2, 2, 64, 32, generator=gen(102)).cuda()
    b = torch.zeros_like(a)
    starts = torch.zeros(3, dtype=torch.int32, device="cuda")
    o = dense.delta_rule(q, k, v, g, beta, a, b, offsets=starts, max_tokens=0)
    torch.cuda.synchronize()
    assert o.shape == (0, 2, 32) and torch.equal(a, b)
    empty = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert dense.delta_rule(q, k, v, g, beta, offsets=empty, max_tokens=5).shape == (0, 2, 32)


def test_refusals():
    q, k, v, g, beta = (x.cuda() for x in delta_inputs(103, [4], 1, 2, 64, 32, BF16))
    pool = torch.zeros(1, 2, 64, 32, device="cuda")
    for bad in (dict(q=q[:, :, :32], k=k[:, :, :32]), dict(k=k[:3]), dict(v=v[:, :, :24]), dict(q=q.float()),
                dict(g=g.double()), dict(beta=beta[:3]), dict(state_in=pool[:, :1]), dict(state_out=pool.double()),
                dict(state_in=pool.transpose(2, 3)), dict(max_tokens=3), dict(scale=float("nan")),
                dict(out=torch.empty(4, 2, 16, device="cuda", dtype=BF16)),
                dict(slots=torch.zeros(2, dtype=torch.int32, device="cuda")),
                dict(offsets=torch.zeros(2, dtype=torch.int64, device="cuda"))):
        with pytest.raises(ValueError):
            dense.delta_rule(**{**dict(q=q, k=k, v=v, g=g, beta=beta), **bad})
