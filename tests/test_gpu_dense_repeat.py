"""A call gives the same bits every time, also beside other work on the card."""
import pytest
import torch

from dense_fixtures import delta_inputs, gen, q4_weights
from fronk_amd import dense

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def repeated(call, times=30):
    want = [t.clone() for t in call()]
    busy = torch.cuda.Stream()
    a, b = torch.empty(1 << 26, device="cuda"), torch.empty(1 << 26, device="cuda")
    busy.wait_stream(torch.cuda.current_stream())
    for i in range(times):
        if i % 3 == 0:
            with torch.cuda.stream(busy):
                b.copy_(a)
        got = call()
        assert all(torch.equal(x, y) for x, y in zip(got, want)), f"call {i}"
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
def test_delta_prompt(dtype):
    q, k, v, g, beta = (x.cuda() for x in delta_inputs(800, [2100], 16, 32, 128, 128, dtype))
    pool = torch.empty(1, 32, 128, 128, device="cuda")
    repeated(lambda: (dense.delta_rule(q, k, v, g, beta, None, pool, normalize=True), pool))


@pytest.mark.parametrize("dtype", [BF16, torch.float16, torch.float32])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_product_of_many_tokens(group, dtype):
    codes, scales, _ = (t.cuda() if t is not None else None for t in q4_weights(801, 4096, 4096, group, False))
    x = torch.randn(512, 4096, generator=gen(802)).to(dtype).cuda()
    repeated(lambda: (dense.q4_product(x, codes, scales),))


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
def test_long_context(dtype):
    n = 40000
    cache = dense.KVCache.empty(n // 64 + 1, 2, 64, 256)
    kv = torch.randn(2, n, 2, 256, device="cuda").to(BF16)
    dense.kv_append(cache, kv[0], kv[1], torch.arange(n, dtype=torch.int32, device="cuda"))
    q = torch.randn(1, 16, 256, generator=gen(803)).to(dtype).cuda()
    table = torch.arange(n // 64 + 1, dtype=torch.int32, device="cuda")[None]
    length = torch.tensor([n], dtype=torch.int32, device="cuda")
    repeated(lambda: (dense.kv_attend(cache, q, table, length),))
