"""What the dense operators write in place, autograd sees; what it would have to
follow is refused."""
import pytest
import torch

from dense_fixtures import delta_inputs, q4_weights
from fronk_amd import dense

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def test_writes_in_place_are_seen():
    q, k, v, g, beta = (x.cuda() for x in delta_inputs(300, [3], 1, 2, 64, 32, BF16))
    pool, out = torch.zeros(1, 2, 64, 32, device="cuda"), torch.empty_like(v)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    codes, scales, _ = q4_weights(301, 8, 64, 32, False)
    x, y = torch.randn(2, 64, device="cuda"), torch.empty(2, 8, device="cuda")
    cache = dense.KVCache.empty(2, 1, 16, 64)
    kv, slots = torch.randn(2, 1, 64, device="cuda"), torch.arange(2, dtype=torch.int32, device="cuda")
    table, lengths = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")
    o = torch.empty(1, 2, 64, device="cuda")

    def raises(f, written, read):
        before, old = [t._version for t in written], [t._version for t in read]
        f()
        assert all(t._version > n for t, n in zip(written, before))
        assert all(t._version == n for t, n in zip(read, old))

    raises(lambda: dense.delta_rule(q, k, v, g, beta, pool, pool, out=out, status=status), [pool, out, status],
           [q, k, v, g, beta])
    codes, scales = codes.cuda(), scales.cuda()
    raises(lambda: dense.q4_product(x, codes, scales, out=y), [y], [x, codes, scales])
    raises(lambda: dense.kv_append(cache, kv, kv, slots, status=status), [*cache, status], [kv, slots])
    raises(lambda: dense.kv_read(cache, slots, status=status), [status], [*cache, slots])
    raises(lambda: dense.kv_attend(cache, kv[:1].expand(1, 2, 64), table, lengths, out=o, status=status), [o, status],
           [*cache, table, lengths])
    # A tensor that a backward pass needs: its change is an error there, not a wrong gradient.
    w = torch.ones(2, 8, device="cuda", requires_grad=True)
    z = (w * y).sum()
    dense.q4_product(x, codes, scales, out=y)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()
    # Inference tensors have no version.
    with torch.inference_mode():
        frozen = torch.empty(2, 8, device="cuda")
    dense.q4_product(x, codes, scales, out=frozen)
    assert torch.equal(frozen, y)


def test_gradients_are_refused():
    codes, scales, _ = q4_weights(302, 8, 64, 32, False)
    x = torch.randn(2, 64, device="cuda", requires_grad=True)
    codes, scales = codes.cuda(), scales.cuda()
    with pytest.raises(ValueError, match="gradient"):
        dense.q4_product(x, codes, scales)
    with torch.no_grad():
        y = dense.q4_product(x, codes, scales)
    assert torch.equal(y, dense.q4_product(x.detach(), codes, scales)) and not y.requires_grad
