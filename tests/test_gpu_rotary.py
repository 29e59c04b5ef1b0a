"""Rotary positions against the formula in 64 bits: both layouts, all or part of a
head, far and negative positions, strides, in place, and graphs."""
import pytest
import torch

from dense_fixtures import HALF, gen, near
from fronk_amd import dense

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def turned(x, positions, f, interleaved, magnitude):
    """(values, tolerance): one rounding of x's type; cosines and sines in fp32 (2^-23
    and half a step, as the angle's turns), two products and a sum; the angle's own 64 bits."""
    angle = positions.double()[:, None] * f.double()
    c, s = magnitude * torch.cos(angle)[:, None], magnitude * torch.sin(angle)[:, None]
    n, y = f.shape[0], x.double().clone()
    at = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    a, b = (x.double()[..., i] for i in at)
    y[..., at[0]], y[..., at[1]] = a * c - b * s, a * s + b * c
    size = torch.zeros_like(y)
    each = magnitude * (2.0 ** -22 + 2.0 ** -51 * angle.abs()[:, None])
    size[..., at[0]] = size[..., at[1]] = each * (a.abs() + b.abs())
    tol = HALF[x.dtype] * y.abs() + size
    tol[..., 2 * n:] = 0
    return y, tol


def make(seed, tokens, heads, kv_heads, dim, dtype):
    r = gen(seed)
    return torch.randn(tokens, heads, dim, generator=r).to(dtype), torch.randn(tokens, kv_heads, dim, generator=r).to(dtype)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,kv_heads,dim,pairs", [
    (1, 16, 2, 256, 32), (37, 4, 1, 128, 64), (300, 3, 3, 64, 32), (5, 1, 1, 2, 1), (9, 2, 1, 80, 37), (7, 5, 2, 96, 24),
    (2, 1, 1, 1024, 512), (3, 2, 2, 1023, 300), (17, 2, 1, 64, 4), (1, 300, 40, 64, 32)])
def test_values(dtype, interleaved, tokens, heads, kv_heads, dim, pairs):
    q, k = make(1, tokens, heads, kv_heads, dim, dtype)
    f, _ = dense.rotary_frequencies(2 * pairs)
    positions = torch.randint(0, 5000, (tokens,), dtype=torch.int32, generator=gen(2))
    a, b = dense.rotary(q.cuda(), k.cuda(), positions.cuda(), f, interleaved=interleaved)
    assert a.dtype == b.dtype == dtype
    near(a, *turned(q, positions, f.cpu(), interleaved, 1.0), "q")
    near(b, *turned(k, positions, f.cpu(), interleaved, 1.0), "k")
    near(dense.rotary(q.cuda(), None, positions.cuda(), f, interleaved=interleaved)[0], *turned(q, positions, f.cpu(), interleaved, 1.0), "q alone")


@pytest.mark.parametrize("interleaved", [False, True])
def test_far_positions(interleaved):
    """Angles of millions of turns, scaled frequencies, a magnitude."""
    places = [0, 1, -1, 131071, 10 ** 6, -10 ** 6, 2 ** 31 - 1, -2 ** 31]
    q, k = make(3, len(places), 2, 1, 64, F32)
    positions = torch.tensor(places, dtype=torch.int32)
    f, m = dense.rotary_frequencies(64, 500000.0, factor=32.0, context=4096)
    assert m > 1.3
    a, b = dense.rotary(q.cuda(), k.cuda(), positions.cuda(), f, interleaved=interleaved, magnitude=m)
    near(a, *turned(q, positions, f.cpu(), interleaved, m), "q")
    near(b, *turned(k, positions, f.cpu(), interleaved, m), "k")


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shift,pairs", [(0, 32), (8, 16), (1, 32), (0, 5)])
def test_strides_and_in_place(dtype, interleaved, shift, pairs):
    """Views of one projection's rows; what is not rotated, and not theirs, stays."""
    tokens, dim = 21, 64
    f, _ = dense.rotary_frequencies(2 * pairs)
    positions = torch.arange(100, 100 + tokens, dtype=torch.int32)
    flat = torch.randn(tokens * (6 * dim + 8) + 16, generator=gen(4)).to(dtype)
    view = lambda t: t[shift:shift + tokens * (6 * dim + 8)].view(tokens, -1)
    parts = lambda t: (view(t)[:, :3 * dim].unflatten(1, (3, dim)), view(t)[:, 3 * dim:5 * dim].unflatten(1, (2, dim)))
    moved = flat.cuda()
    q, k = parts(moved)
    out = torch.full((tokens, 7, dim + 8), 3.0, dtype=dtype, device="cuda")
    places = out[:, :3, shift:shift + dim] if shift else out[:, :3, :dim], out[:, 4:6, :dim]
    a, b = dense.rotary(q, k, positions.cuda(), f, interleaved=interleaved, out=places)
    assert a.data_ptr() == places[0].data_ptr() and torch.equal(moved.cpu(), flat)
    want = [turned(x, positions, f.cpu(), interleaved, 1.0) for x in parts(flat)]
    near(a, *want[0], "q"), near(b, *want[1], "k")
    places[0].fill_(3.0), places[1].fill_(3.0)
    assert (out == 3.0).all()
    dense.rotary(q, k, positions.cuda(), f, interleaved=interleaved, out=(q, k))
    after = moved.cpu()
    for got, x in zip(parts(after), want):
        near(got, *x, "in place")
    for x, y in zip(parts(after), parts(flat)):
        x.copy_(y)
    assert torch.equal(after, flat)
    # One of the two in place, the other apart.
    moved.copy_(flat)
    dense.rotary(q, k, positions.cuda(), f, interleaved=interleaved, out=(q, places[1]))
    near(q, *want[0], "q in place"), near(places[1], *want[1], "k apart")
    assert torch.equal(k.cpu(), parts(flat)[1])


def test_values_that_are_not_finite_stay_in_their_pair():
    q, k = make(5, 4, 2, 1, 64, BF16)
    q[1, 0, 3] = float("inf")
    f, _ = dense.rotary_frequencies(64)
    positions = torch.arange(4, dtype=torch.int32)
    got, _ = dense.rotary(q.cuda(), k.cuda(), positions.cuda(), f)
    hit = torch.zeros(4, 2, 64, dtype=torch.bool)
    hit[1, 0, 3] = hit[1, 0, 35] = True
    assert torch.equal(torch.isfinite(got.cpu()), ~hit)


def test_refusals():
    q, k = (x.cuda() for x in make(6, 3, 2, 1, 64, BF16))
    f, _ = dense.rotary_frequencies(64)
    p = torch.arange(3, dtype=torch.int32, device="cuda")
    for args, kw in (((q, k, p.long(), f), {}), ((q, k, p[:2], f), {}), ((q, k, p, f.float()), {}), ((q, k, p, f[:0]), {}),
                     ((q, k, p, torch.cat([f, f])), {}), ((q, k[:2], p, f), {}), ((q, k.float(), p, f), {}), ((q, k[..., :32], p, f), {}),
                     ((q, k, p, f), dict(out=q)), ((q, k, p, f), dict(out=(q, q[:, :1]))), ((q, k, p, f), dict(out=(q[:1].expand(3, 2, 64), k))),
                     ((q, k, p, f), dict(magnitude=float("nan"))), ((q, None, p, f), dict(out=(q, k))), ((q, k, p.cpu(), f), {}),
                     ((q[..., ::2], k[..., ::2], p, f[:16]), {}), ((q[:2], k[:2], p[:2], f), dict(out=(q[1:], k[1:]))),
                     ((q, k, p, f[None]), {})):
        with pytest.raises(ValueError):
            dense.rotary(*args, **kw)
    with pytest.raises(ValueError, match="gradient"):
        dense.rotary(q.float().requires_grad_(), None, p, f)
    assert dense.rotary(q[:0], k[:0], p[:0], f)[0].shape == (0, 2, 64)
    before = q._version, k._version, p._version
    dense.rotary(q, k, p, f, out=(q, k))
    assert q._version > before[0] and k._version > before[1] and p._version == before[2]


def test_replays():
    q, k = make(7, 5, 4, 2, 128, F16)
    a, b = q.cuda(), k.cuda()
    f, _ = dense.rotary_frequencies(128)
    p = torch.arange(5, dtype=torch.int32, device="cuda")
    dense.rotary(a, b, p, f)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        x, y = dense.rotary(a, b, p, f)
    for step in range(3):
        p.add_(1000)
        g.replay()
        torch.cuda.synchronize()
        near(x, *turned(q, p.cpu(), f.cpu(), False, 1.0), "q")
        assert torch.equal(y, dense.rotary(a, b, p, f)[1])
