"""The dense operators at the sizes that send them other ways than the rest of
their tests: many chunks, many streams, wide values, long rows, long contexts and
as many tokens as there may be."""
import pytest
import torch

import test_gpu_delta
import test_gpu_kv
import test_gpu_q4

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("lens,key_heads,heads,dk,dv", [
    ([1000, 1, 777, 0, 64, 1300, 129, 900], 8, 24, 64, 16), ([4100], 6, 24, 64, 32), ([300] * 20, 4, 16, 128, 16),
    ([33, 500] * 6, 16, 32, 64, 16)])
def test_value_heads_that_share_a_workgroup(lens, key_heads, heads, dk, dv, dtype):
    """1536 workgroups and more, were there one for each head's chunk."""
    assert (sum(lens) // 64 + len(lens)) * heads >= 1536
    test_gpu_delta.compare(500, lens, key_heads, heads, dk, dv, dtype, True)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dv", [32, 48, 64, 80, 112])
def test_streams_that_fill_the_card(dv, dtype):
    """Several tiles of 16 columns a workgroup, the last one not whole."""
    lens = [i % 5 for i in range(150)]
    assert len(lens) * 4 * dv // 16 > 1024
    test_gpu_delta.compare(501, lens, 2, 4, 64, dv, dtype, True)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("dk,dv", [(64, 256), (128, 1024), (256, 528)])
def test_wide_values(dk, dv, dtype):
    test_gpu_delta.compare(502, [3, 1], 1, 2, dk, dv, dtype, True)
    test_gpu_delta.compare(503, [70, 5], 1, 2, dk, dv, dtype, True)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("lens,burst,heads,kv_heads", [([9000], 1, 4, 1), ([20001], 3, 8, 1), ([17000, 40, 8500], 1, 2, 2)])
def test_contexts_of_many_stretches(lens, burst, heads, kv_heads, dim, dtype):
    """More than 32 of them are joined by slices of a row."""
    test_gpu_kv.compare(504, lens, burst, heads, kv_heads, 64, dim, dtype)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("tokens,cols,rows,group", [(1, 65536, 33, 64), (5, 65536, 17, 128), (20, 65536, 50, 32),
                                                    (100, 65536, 300, 128), (70, 40960, 500, 32)])
def test_long_rows(tokens, cols, rows, group, dtype):
    test_gpu_q4.compare(505, tokens, cols, rows, group, dtype, True)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("tokens,cols,rows,group", [(4096, 256, 2000, 64), (4096, 128, 200, 128), (1000, 384, 3000, 128),
                                                    (3, 256, 66000, 64), (90, 128, 66000, 32)])
def test_many_tokens_and_rows(tokens, cols, rows, group, dtype):
    test_gpu_q4.compare(506, tokens, cols, rows, group, dtype)
