"""The gated delta rule over more sequences than a wavefront looks through by
itself: their order, and bad ones among them."""
import pytest
import torch

from dense_fixtures import delta, delta_inputs, delta_tolerance, gen, near
from fronk_amd import dense

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def lengths(n, most, seed):
    """Mostly none and one, a few up to `most`."""
    x = torch.randint(0, 2, (n,), generator=gen(seed))
    x[::97] = torch.randint(0, most + 1, (len(x[::97]),), generator=gen(seed + 1))
    x[n // 2] = most
    return x.tolist()


@pytest.mark.parametrize("most", [3, 70])
@pytest.mark.parametrize("n", [2049, 4097, 9001])
def test_many(n, most):
    lens = lengths(n, most, 400)
    q, k, v, g, beta = delta_inputs(402, lens, 1, 1, 64, 16, F32)
    state = torch.randn(n, 1, 64, 16, generator=gen(403))
    want, final = delta(q, k, v, g, beta, state, lens, 0.125, True)
    starts = torch.cat([torch.zeros(1, dtype=torch.int64), torch.tensor(lens).cumsum(0)]).to(torch.int32).cuda()
    pool, status = state.cuda(), torch.zeros(1, dtype=torch.int32, device="cuda")
    o = dense.delta_rule(*(x.cuda() for x in (q, k, v, g, beta)), pool, pool, scale=0.125, offsets=starts,
                         max_tokens=most, normalize=True, status=status)
    assert status.item() == 0
    size = max(float(final.abs().max()), 1.0)
    near(o, want, delta_tolerance(want, F32, 64, most, size), "o")
    near(pool, final, delta_tolerance(final, F32, 64, most, size), "state")


@pytest.mark.parametrize("most", [2, 64])
@pytest.mark.parametrize("at", [1, 255, 4095, 4096, 5000])
def test_offsets_that_go_down_among_many(at, most):
    """What begins below an offset before it is left out, also thousands on."""
    n, total = 6000, 6000
    starts = torch.arange(n + 1, dtype=torch.int32)
    starts[at] = at + 2          # its sequence is of one token less than none: bad; the next begins below
    q, k, v, g, beta = (x.cuda() for x in delta_inputs(404, [total], 1, 1, 64, 16, BF16))
    pool = torch.randn(n, 1, 64, 16, generator=gen(405)).cuda()
    good = pool.clone()
    o = dense.delta_rule(q, k, v, g, beta, good, good, offsets=torch.arange(n + 1, dtype=torch.int32).cuda(),
                         max_tokens=most, normalize=True)
    p, out = pool.clone(), torch.full_like(v, 3.0)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    dense.delta_rule(q, k, v, g, beta, p, p, offsets=starts.cuda(), max_tokens=1 if most == 2 else most, out=out,
                     normalize=True, status=status)
    assert status.item() == dense.BAD_OFFSET
    bad = torch.zeros(n, dtype=torch.bool)
    begins, seen = starts[:-1].long(), torch.cummax(torch.cat([torch.tensor([-1]), starts[:-2].long()]), 0).values
    long = starts[1:] - starts[:-1] > (1 if most == 2 else most)
    bad |= (begins < seen) | (starts[1:] < starts[:-1]) | long
    assert 1 <= bad.sum() <= 3
    assert torch.equal(p[bad], pool[bad])
    # Those of the very tokens they had before.
    same = ~bad & (starts[:-1] == torch.arange(n)) & (starts[1:] == torch.arange(1, n + 1))
    assert same.sum() >= n - 4 and torch.equal(p[same], good[same]) and torch.equal(out[same], o[same])


def test_many_in_a_graph():
    n = 2100
    q, k, v, g, beta = (x.cuda() for x in delta_inputs(406, [1] * n, 1, 1, 64, 16, BF16))
    first = torch.randn(n, 1, 64, 16, generator=gen(407)).cuda()
    starts, pool = torch.arange(n + 1, dtype=torch.int32).cuda(), first.clone()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    kw = dict(offsets=starts, max_tokens=1, normalize=True, status=status)
    eager = first.clone()
    want = dense.delta_rule(q, k, v, g, beta, eager, eager, **kw)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = dense.delta_rule(q, k, v, g, beta, pool, pool, **kw)
    for down in (False, True, False):
        pool.copy_(first), status.zero_(), starts.copy_(torch.arange(n + 1))
        if down:
            starts[500] = 400
        graph.replay()
        torch.cuda.synchronize()
        assert status.item() == (dense.BAD_OFFSET if down else 0)
        if down:
            assert torch.equal(pool[:499], eager[:499]) and torch.equal(pool[500], first[500])
        else:
            assert torch.equal(o, want) and torch.equal(pool, eager)
        torch.cuda.synchronize()
