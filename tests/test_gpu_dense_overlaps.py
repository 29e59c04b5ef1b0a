"""Outputs in places that other workgroups read, or in one place, are refused."""
import pytest
import torch

from dense_fixtures import delta_inputs, q4_weights
from fronk_amd import dense

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def test_delta_outputs():
    q, k, v, g, beta = (x.cuda() for x in delta_inputs(700, [4], 2, 2, 64, 64, BF16))
    args = dict(q=q, k=k, v=v, g=g, beta=beta)
    for out in (q, k, v, v.clone()[:1].expand(4, 2, 64), q.view(4, 2, 64)):
        with pytest.raises(ValueError, match="out"):
            dense.delta_rule(**args, out=out)
    # Views of one buffer that share nothing.
    buffer = torch.empty(4, 4, 64, dtype=BF16, device="cuda")
    buffer[:, :2] = v
    want = dense.delta_rule(**args)
    args["v"] = buffer[:, :2]
    assert torch.equal(dense.delta_rule(**args, out=buffer[:, 2:]), want)
    # Pools that share some of their rows.
    pool = torch.zeros(3, 2, 64, 64, device="cuda")
    two = {n: torch.cat([t, t]) for n, t in args.items()}
    with pytest.raises(ValueError):
        dense.delta_rule(**two, max_tokens=4, state_in=pool[:2], state_out=pool[1:])
    dense.delta_rule(**two, max_tokens=4, state_in=pool[:2], state_out=pool[:2])


def test_product_outputs():
    codes, scales, _ = (t.cuda() if t is not None else None for t in q4_weights(701, 64, 64, 32, False))
    x = torch.randn(5, 64, device="cuda").to(BF16)
    for out in (x, x[:1].expand(5, 64), x.view(5, 64)):
        with pytest.raises(ValueError, match="out"):
            dense.q4_product(x, codes, scales, out=out)
    with pytest.raises(ValueError, match="out"):
        dense.q4_product(x[:4], codes, scales, out=x[1:])
    wide = torch.randn(5, 128, device="cuda").to(BF16)
    want = dense.q4_product(wide[:, :64].clone(), codes, scales)
    assert torch.equal(dense.q4_product(wide[:, :64], codes, scales, out=wide[:, 64:]), want)


def test_attention_outputs():
    cache = dense.KVCache.empty(1, 1, 16, 64)
    kv = torch.randn(4, 1, 64, device="cuda")
    dense.kv_append(cache, kv, kv, torch.arange(4, dtype=torch.int32, device="cuda"))
    q, table = torch.randn(2, 2, 64, device="cuda"), torch.zeros(2, 1, dtype=torch.int32, device="cuda")
    length = torch.tensor([4, 3], dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="out"):
        dense.kv_attend(cache, q, table, length, out=q[:1].expand(2, 2, 64))
