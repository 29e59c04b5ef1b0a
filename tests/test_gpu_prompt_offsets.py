"""Keys' offsets of prompts are held to the same order as the queries'."""
import pytest
import torch

from dense_fixtures import gen
from fronk_amd import dense

pytestmark = pytest.mark.gpu


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 64), (torch.float16, 128), (torch.float32, 256)])
@pytest.mark.parametrize("context", [60, 5000])
@pytest.mark.parametrize("with_offsets", [True, False])
def test_keys_that_begin_below_earlier_ones(with_offsets, context, dtype, dim):
    """A sequence that ends below its start is bad, and one that begins below an offset before it too,
    whichever offsets are given; few rows over many keys go in stretches, whose join sees the same."""
    r = gen(50)
    q, k, v = (torch.randn(n, h, dim, generator=r).to(dtype).cuda() for n, h in ((60, 2), (context, 1), (context, 1)))
    status, kw = torch.zeros(1, dtype=torch.int32, device="cuda"), dict(max_tokens=20, max_context=context)
    if with_offsets:
        kw["offsets"] = ints([0, 20, 40, 60])

    def run(k_offsets):
        out = torch.full_like(q, 9.0)
        status.zero_()
        dense.prompt_attend(q, k, v, k_offsets=ints(k_offsets), out=out, status=status, **kw)
        return out, status.item()

    last = context
    want, bad = run([0, 20, 30, last])
    assert bad == 0
    for k_offsets, good in (([0, 30, 10, last], [0]), ([40, 20, 30, last], []), ([5, 0, 4, 10], []), ([0, 20, 20, 10], [0, 1]),
                            ([0, 20, 30, last], [0, 1, 2])):
        got, bad = run(k_offsets)
        assert bad == (0 if len(good) == 3 else dense.BAD_OFFSET), k_offsets
        for i in range(3):
            part = got[20 * i:20 * i + 20]
            assert bool((part == 9.0).all()) == (i not in good), (k_offsets, i)
        if 0 in good and k_offsets[1] == 20:
            assert torch.equal(got[:20], want[:20])
