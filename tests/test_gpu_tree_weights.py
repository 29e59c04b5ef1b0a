"""Weights of draft trees in two or more parts, as kv_attend has them over the same cache: a
burst that becomes a chain of drafts loses no bits."""
import pytest
import torch

from attention_fixtures import softmax_rows
from dense_fixtures import HALF, U, gen, near
from fronk_amd import dense

pytestmark = pytest.mark.gpu

# Two bf16 parts leave 2^-16 of a weight; fp32's third one 2^-24.
PARTS = {torch.bfloat16: 2.0 ** -16, torch.float16: 2.0 ** -16, torch.float32: 2.0 ** -23}


@pytest.mark.parametrize("dtype", list(PARTS))
@pytest.mark.parametrize("heads,kv_heads,dim,length,drafts", [(4, 1, 64, 300, 8), (8, 2, 128, 700, 5), (4, 2, 256, 500, 8), (16, 1, 128, 4000, 3),
                                                              (8, 1, 256, 1000, 8)])
def test_chains_and_bursts(heads, kv_heads, dim, length, drafts, dtype):
    """What is held, its values with signs that nearly cancel, against 64 bits: a chain's error is the outputs' rounding,
    fp32's and the parts', and the burst's is no less."""
    r, page = gen(40), 32
    pages = (length + page - 1) // page
    cache = dense.KVCache.empty(pages, kv_heads, page, dim)
    k, v = torch.randn(length, kv_heads, dim, generator=r), torch.randn(length, kv_heads, dim, generator=r).abs() + 4
    v[1::2] *= -1
    slots = torch.arange(length, dtype=torch.int32, device="cuda")
    dense.kv_append(cache, k.cuda(), v.cuda(), slots)
    k, v = (x.cpu() for x in dense.kv_read(cache, slots, torch.float32))
    q = torch.randn(drafts, heads, dim, generator=r).to(dtype)
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
    n = torch.tensor([length], dtype=torch.int32, device="cuda")
    chain = torch.tensor([(2 << b) - 1 for b in range(drafts)], device="cuda")
    seen = torch.arange(length) <= length - drafts + torch.arange(drafts)[:, None]
    o, size, terms = softmax_rows(q, k, v, seen, dim ** -0.5)
    delta = U * ((dim + 2) * terms + length) + 2.0 ** -22
    tol = HALF[dtype] * o.abs() + (PARTS[dtype] + 2 * delta) * size
    near(dense.kv_attend(cache, q.cuda(), table, n), o, tol, "burst")
    near(dense.kv_attend_tree(cache, q.cuda(), chain, table, n), o, tol, "chain")
