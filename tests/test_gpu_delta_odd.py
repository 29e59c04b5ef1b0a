"""The gated delta rule where a chunk's factored form leaves fp32 or meets
numbers that are none: growing states, magnitudes next to the largest, and
infinities and NaN, which reach no token before theirs. As in test_gpu_delta.py,
n up to 32 goes token by token and above in chunks."""
import pytest
import torch

from dense_fixtures import HALF, U, delta_inputs, gen
from fronk_amd import dense

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
NAN, INF = float("nan"), float("inf")


def walk(q, k, v, g, beta, state, scale, normalize):
    """(o, states after each token) in 64 bits; one sequence, state [heads][dk][dv]."""
    q, k, v, g, beta, s = (x.double() for x in (q, k, v, g, beta, state))
    if normalize:
        q, k = (x / (x.square().sum(-1, keepdim=True) + 1e-6).sqrt() for x in (q, k))
    r = v.shape[1] // q.shape[1]
    q, k = q.repeat_interleave(r, 1), k.repeat_interleave(r, 1)
    o, states = torch.zeros_like(v), [s]
    for t in range(v.shape[0]):
        s = s * torch.exp(g[t])[:, None, None]
        u = beta[t][:, None] * (v[t] - (s * k[t][..., None]).sum(1))
        s = s + k[t][..., None] * u[:, None, :]
        o[t] = scale * (s * q[t][..., None]).sum(1)
        states.append(s)
    return o, torch.stack(states)


def grown(states, g, v):
    """[heads]: the largest that a number which is rounded on the way (a state's or
    an update's, for values v) becomes by the decays behind it."""
    top = states.abs().amax((2, 3))
    top[1:] = torch.maximum(top[1:], v.double().abs().amax(2))
    total = torch.cat([torch.zeros(1, g.shape[1], dtype=torch.float64), torch.cumsum(g.double(), 0)])
    best = torch.full(top.shape[1:], -INF, dtype=torch.float64)
    most = torch.zeros_like(best)
    for t in range(len(top)):
        best = torch.maximum(best, torch.log(top[t]) - total[t])
        most = torch.maximum(most, torch.exp(best + total[t]))
    return most


def call(q, k, v, g, beta, state, scale, normalize):
    pool = state[None].cuda()
    o = dense.delta_rule(*(x.cuda() for x in (q, k, v, g, beta)), pool, pool, scale=scale, normalize=normalize)
    return o.cpu(), pool[0].cpu()


def close(got, want, tol, what):
    off = (got.double() - want).abs() - tol
    assert torch.isfinite(got).all() and off.max() <= 0, f"{what}: {off.max():.3g} over its tolerance"


def compare(q, k, v, g, beta, state, normalize=True):
    """Against 64 bits; rounding errors grow and shrink as the states do: a random
    walk over n tokens of sums over dk terms, eight standard deviations of it."""
    n, dk = v.shape[0], q.shape[2]
    want, states = walk(q, k, v, g, beta, state, 0.125, normalize)
    size = grown(states, g, v)
    o, final = call(q, k, v, g, beta, state, 0.125, normalize)
    tol = 8 * U * (dk * (n + 1)) ** 0.5 * size
    close(o, want, HALF[v.dtype] * want.abs() + tol[None, :, None], "o")
    close(final, states[-1], tol[:, None, None], "state")


@pytest.mark.parametrize("n", [4, 130])
def test_large_growth_from_nothing(n):
    """e^g that only zeros meet, then growth that passes fp32 within a chunk if it
    is taken by itself."""
    q, k, v, g, beta = delta_inputs(200, [n], 1, 2, 64, 32, F32)
    g[0], g[1] = 80.0, 10.0
    compare(q, k, v, g, beta, torch.zeros(2, 64, 32))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("n", [20, 130, 300])
def test_slow_growth(n, dtype):
    q, k, v, g, beta = delta_inputs(201, [n], 2, 4, 64, 32, dtype)
    g[:, :2] = 0.01 * torch.rand(n, 2, generator=gen(202))
    compare(q, k, v, g, beta, torch.randn(4, 64, 32, generator=gen(203)))


@pytest.mark.parametrize("growth", [0.02, 0.1, 0.3])
@pytest.mark.parametrize("n", [30, 64, 100])
def test_growth_that_each_token_takes_back(n, growth):
    """One key for all tokens and beta 1: what has grown is replaced by the next
    value. (Rounding errors beside the key are not, and grow.)"""
    q, k, v, g, beta = delta_inputs(220, [n], 1, 1, 64, 16, F32)
    k[:] = k[0]
    g[:], beta[:] = growth, 1.0
    compare(q, k, v, g, beta, torch.zeros(1, 64, 16))


@pytest.mark.parametrize("first", [0, 70])
def test_small_states_that_grow_past_a_chunks_factors(first):
    """Values near 1e-25 that grow by e^120 within thirty tokens and shrink again."""
    n = 200
    q, k, v, g, beta = delta_inputs(204, [n], 1, 3, 64, 16, F32)
    v *= 1e-25
    g[:] = 0.0
    g[first:first + 30, 0], g[first + 30:first + 60, 0] = 4.0, -4.0
    g[first:first + 2, 1], g[first + 2:first + 4, 1] = 59.0, -60.0
    compare(q, k, v, g, beta, 1e-25 * torch.randn(3, 64, 16, generator=gen(205)))


@pytest.mark.parametrize("n", [3, 100])
def test_decay_and_growth_between_two_tokens(n):
    """A state emptied by -100 and one token's growth of as much right behind it."""
    q, k, v, g, beta = delta_inputs(206, [n], 1, 2, 64, 32, F32)
    g[:] = 0.0
    g[1], g[2] = -100.0, 80.0
    v[1] = 0.0
    v[0] *= 1e-3
    compare(q, k, v, g, beta, torch.randn(2, 64, 32, generator=gen(207)))


@pytest.mark.parametrize("n", [3, 100])
def test_magnitudes_next_to_the_largest(n):
    """A value above bf16's largest, and a state with a row of 2e38."""
    q, k, v, g, beta = delta_inputs(208, [n], 1, 2, 64, 32, F32, False)
    q *= 0.1
    g[:], beta[:] = -1.0, 1e-3
    v[:] = 0.5
    v[n // 2, 0] = 3.395e38
    state = torch.zeros(2, 64, 32)
    state[1, 5] = 2e38 * torch.sign(torch.randn(32, generator=gen(209)))
    compare(q, k, v, g, beta, state, False)


PLACES = [(4, 0), (4, 2), (130, 0), (130, 31), (130, 63), (130, 64), (130, 129), (200, 100)]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("value", [INF, -INF, NAN])
@pytest.mark.parametrize("n,t", PLACES)
def test_a_non_finite_value(n, t, value, dtype):
    """v of one token, head and column: that column from the token on."""
    q, k, v, g, beta = delta_inputs(210, [n], 2, 4, 64, 48, dtype)
    state = torch.randn(4, 64, 48, generator=gen(211))
    want, states = walk(q, k, v, g, beta, state, 0.125, True)
    tol = 8 * U * (64 * (n + 1)) ** 0.5 * max(float(states.abs().max()), 1.0)
    v = v.clone()
    v[t, 1, 20] = value
    o, final = call(q, k, v, g, beta, state, 0.125, True)
    hit = torch.zeros(n, 4, 48, dtype=torch.bool)
    hit[t:, 1, 20] = True
    assert not torch.isfinite(o[hit]).any() and not torch.isfinite(final[1, :, 20]).any()
    close(o[~hit], want[~hit], HALF[dtype] * want[~hit].abs() + tol, "o")
    rest = torch.ones(4, 48, dtype=torch.bool)
    rest[1, 20] = False
    close(final.transpose(1, 2)[rest], states[-1].transpose(1, 2)[rest], tol, "state")


@pytest.mark.parametrize("what", ["k", "beta", "g"])
@pytest.mark.parametrize("value", [INF, NAN])
@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("n,t", PLACES)
def test_a_non_finite_key_or_gate(n, t, normalize, value, what):
    """The heads that it reaches, from its token on."""
    dtype = F32 if what == "k" else BF16
    q, k, v, g, beta = delta_inputs(212, [n], 2, 4, 64, 32, dtype, normalize)
    state = torch.randn(4, 64, 32, generator=gen(213))
    want, states = walk(q, k, v, g, beta, state, 0.125, normalize)
    tol = 8 * U * (64 * (n + 1)) ** 0.5 * max(float(states.abs().max()), 1.0)
    if what == "k":
        k = k.clone()
        k[t, 1, 7], heads = value, [2, 3]
    else:
        (beta if what == "beta" else g)[t, 2], heads = value, [2]
    o, final = call(q, k, v, g, beta, state, 0.125, normalize)
    hit = torch.zeros(n, 4, dtype=torch.bool)
    hit[t:, heads] = True
    left = [h for h in range(4) if h not in heads]
    assert not torch.isfinite(o[hit]).any()
    # (an infinite key reaches the rows of the state that it has a part in)
    assert not torch.isfinite(final[heads]).all((1, 2)).any()
    scale = 8.0 if not normalize else 1.0   # |q| of some sqrt(dk)
    close(o[~hit], want[~hit], HALF[dtype] * want[~hit].abs() + scale * tol, "o")
    close(final[left], states[-1][left], tol, "state")


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("value", [INF, NAN])
@pytest.mark.parametrize("n,t", PLACES)
def test_a_non_finite_query(n, t, value, dtype):
    """Its own outputs only."""
    q, k, v, g, beta = delta_inputs(214, [n], 2, 4, 64, 32, dtype)
    state = torch.randn(4, 64, 32, generator=gen(215))
    want, states = walk(q, k, v, g, beta, state, 0.125, True)
    tol = 8 * U * (64 * (n + 1)) ** 0.5 * max(float(states.abs().max()), 1.0)
    q = q.clone()
    q[t, 0, 3] = value
    o, final = call(q, k, v, g, beta, state, 0.125, True)
    hit = torch.zeros(n, 4, dtype=torch.bool)
    hit[t, :2] = True
    assert not torch.isfinite(o[hit]).any()
    close(o[~hit], want[~hit], HALF[dtype] * want[~hit].abs() + tol, "o")
    close(final, states[-1], tol, "state")


def test_other_sequences_keep_their_bits():
    """And a state that is not finite, in a batch."""
    lens = [70, 40, 100]
    q, k, v, g, beta = (x.cuda() for x in delta_inputs(216, lens, 1, 2, 64, 32, BF16))
    pool = torch.randn(3, 2, 64, 32, generator=gen(217)).cuda()
    starts = torch.tensor([0, 70, 110, 210], dtype=torch.int32).cuda()
    clean, bad = pool.clone(), pool.clone()
    want = dense.delta_rule(q, k, v, g, beta, clean, clean, offsets=starts, max_tokens=100, normalize=True)
    v2 = v.clone()
    v2[75] = INF
    bad[2, 1, 5, 3] = NAN
    before = bad.clone()
    o = dense.delta_rule(q, k, v2, g, beta, bad, bad, offsets=starts, max_tokens=100, normalize=True)
    assert torch.equal(o[:70], want[:70]) and torch.equal(bad[0], clean[0])
    assert torch.isfinite(o[70:75]).all() and not torch.isfinite(o[75:110]).any()
    assert not torch.isfinite(o[110:, 1, 3]).any() and torch.equal(o[110:, 0], want[110:, 0])
    # The same call token by token from there: the same tokens are finite.
    again = dense.delta_rule(q, k, v2, g, beta, before, None, offsets=starts, max_tokens=100, normalize=True)
    assert torch.equal(torch.isfinite(again), torch.isfinite(o))

