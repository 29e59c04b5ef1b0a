"""Weights of prompt attention: those far below a row's largest, which in fp16 would
leave the range of a half, one after the other in every order, and the bits that
weights keep beside the outputs' own rounding."""
import math

import pytest
import torch

from attention_fixtures import prompt
from dense_fixtures import HALF, U, gen, near
from fronk_amd import dense

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def lines(scores, heads, dim, rows, dtype):
    """q and k whose products are `scores` (each exact in fp16 and bf16, as 2 of its parts)."""
    q, k = torch.zeros(rows, heads, dim), torch.zeros(len(scores), 1, dim)
    s = torch.tensor(scores)
    q[:, :, :2] = 1.0
    k[:, 0, 0] = s.to(dtype).float()
    k[:, 0, 1] = (s - k[:, 0, 0]).to(dtype).float()
    return q.to(dtype), k.to(dtype)


def check(q, k, v, weights, scale=1.0, tile=0.0, aligned=True):
    """Outputs against 64 bits: their own rounding (fp16: at least half of 2^-24), `weights`
    of each weight, fp32's share as attend_tolerance has it, and of the largest value `tile`
    and, for each key, the 2^-126 below which an exponential in 32 bits is zero."""
    at = torch.zeros(q.numel() + 8, dtype=q.dtype, device="cuda")[8 if aligned else 1:][:q.numel()].view(q.shape)
    got = dense.prompt_attend(at.copy_(q), k.cuda(), v.cuda(), scale=scale)
    tile += k.shape[0] * 2.0 ** -126
    o, size, terms = prompt(q, k, v, [q.shape[0]], [k.shape[0]], scale)
    delta = U * ((q.shape[2] + 2) * terms + k.shape[0]) + 2.0 ** -22
    own = HALF[q.dtype] * o.abs()
    if q.dtype == F16:
        own = own.clamp(min=2.0 ** -25)
    near(got, o, own + (weights + 2 * delta) * size + tile * v.abs().max().item(), "o")


# A tile has at most 64 keys. In fp16 a weight is off by up to 2^-25 beside its rounding. Where
# the largest of a tile is set to 2^7 and stays (one key above all others), that is 64
# 2^-32 of it for all of the tile's, and no more of the row's sum, as each tile's largest is in it.
TILE = {F16: 64 * 2.0 ** -32, BF16: 0.0, F32: 0.0}
WEIGHT = {F16: HALF[F16], BF16: HALF[BF16], F32: 2.0 ** -22}


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("below", [9.0, 13.0, 17.0, 18.0, 20.0, 25.0, 41.0])
@pytest.mark.parametrize("dim,rows", [(64, 1), (128, 40), (256, 3)])
def test_one_key_far_above_thousands(dim, rows, below, dtype):
    """A first key whose value is zero, as a sink, before 8192 others of one score."""
    m = 8192 + rows
    q, k = lines([20.0] + [20.0 - below] * (m - 1), 2, dim, rows, dtype)
    v = torch.randn(m, 1, dim, generator=gen(30)).abs()
    v[0], v[1:, :, ::2] = 0.0, 1.0
    v = v.to(dtype)
    check(q, k, v, WEIGHT[dtype], tile=TILE[dtype])
    # The other way round: the last of the keys that all rows see.
    at = m - rows
    k[0], k[at], v[0], v[at] = k[at], k[0].clone(), v[at], v[0].clone()
    check(q, k, v, WEIGHT[dtype], tile=TILE[dtype])


# (Any order: a tile's largest weight is at least 1 where 2^-25 is what a weight is off by.)
ORDER = {F16: 64 * 2.0 ** -25, BF16: 0.0, F32: 0.0}


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("below", [9.0, 17.0, 18.0, 25.0])
def test_one_key_far_above_thousands_in_one_stretch(dim, below, dtype):
    """The same where there are as many key heads (one, seen 512 times) as leave no stretches."""
    m = 8192
    q, k = lines([20.0] + [20.0 - below] * (m - 1), 1, dim, 3, dtype)
    v = torch.ones(m, 1, dim, dtype=dtype)
    v[0] = 0.0
    got = dense.prompt_attend(*(x.cuda().expand(x.shape[0], 512, dim) for x in (q, k, v)), scale=1.0)
    assert (got == got[:, :1]).all()
    o, size, terms = prompt(q, k, v, [3], [m], 1.0)
    delta = U * ((dim + 2) * terms + m) + 2.0 ** -22
    own = (HALF[dtype] * o.abs()).clamp(min=2.0 ** -25 if dtype == F16 else 0.0)
    near(got[:, :1], o, own + (WEIGHT[dtype] + 2 * delta) * size + TILE[dtype], "o")


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("step", [0.25, 1.0, 3.0, 8.0])
def test_falling_and_rising_scores(step, dtype):
    """Scores that fall, and rise again above all before: sums are carried down and up, and
    no further than their range."""
    down = [-step * i for i in range(200)]
    q, k = lines(down + down[::-1] + [step * i for i in range(20)], 2, 64, 150, dtype)
    v = torch.randn(k.shape[0], 1, 64, generator=gen(31)).to(dtype)
    check(q, k, v, WEIGHT[dtype], tile=ORDER[dtype])
    check(q, -k, v, WEIGHT[dtype], scale=-1.0, tile=ORDER[dtype])
    # The largest values beside the smallest weights.
    v[:30], v[150:250] = 0.0, 60000.0
    check(q, k, v, WEIGHT[dtype], tile=ORDER[dtype])


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_stretches_of_unlike_scores(dtype):
    """One row over 4096 keys, whose stretches' largest scores differ by much or have nothing to add."""
    r = gen(32)
    scores = [12.0 * math.sin(i / 500) + x for i, x in enumerate(torch.randn(4096, generator=r).tolist())]
    q, k = lines(scores, 4, 128, 1, dtype)
    v = torch.randn(4096, 1, 128, generator=r).to(dtype)
    check(q, k, v, WEIGHT[dtype], tile=ORDER[dtype])


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("aligned", [True, False])
def test_rows_that_see_nothing_of_a_tile(dtype, aligned):
    """Tiles that some rows do not see, behind a key far above the others."""
    n = 300
    q, k = lines([15.0] + [0.0] * (n - 1), 3, 64, n, dtype)
    v = torch.rand(n, 1, 64, generator=gen(33))
    v[0] = 0.0
    v = v.to(dtype)
    check(q, k, v, WEIGHT[dtype], tile=ORDER[dtype], aligned=aligned)


# In two parts a weight is off by the square of a rounding: 2^-16 in bf16; in fp16 the second part
# leaves at most 2^-25 as above.
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("heads,kv_heads,dim,n,m", [(4, 2, 64, 130, 130), (4, 1, 128, 70, 500), (2, 1, 256, 200, 200), (2, 2, 128, 4, 3000)])
def test_weights_keep_their_bits(heads, kv_heads, dim, n, m, dtype):
    r = gen(34)
    q, k, v = (torch.randn(t, h, dim, generator=r).to(dtype) for t, h in ((n, heads), (m, kv_heads), (m, kv_heads)))
    check(q, k, v, HALF[dtype] ** 2, scale=dim ** -0.5, tile=ORDER[dtype])
    # Signs that nearly cancel: outputs are small beside their values.
    v = (v.abs() + 4).to(dtype)
    v[1::2] *= -1
    check(q, k, v, HALF[dtype] ** 2, scale=dim ** -0.5, tile=ORDER[dtype])
