"""Products with 4-bit weights on the GPU against the formula in 64 bits."""
import pytest
import torch

from dense_fixtures import HALF, U, gen, near, q4, q4_weights
from fronk_amd import dense

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def tolerance(want, size, dtype, cols, group):
    """One rounding of the output, and fp32 sums of `size` in magnitude: codes
    and zero points of 32 columns enter two sums, then come the groups' products
    and the partial sums of up to 16 wavefronts, each a rounding of half a step
    (and an internal one of the 32 products)."""
    return HALF[dtype] * want.abs() + (4 * (cols // 32) + 2 * (cols // group) + 16) * U * size


def compare(seed, tokens, cols, rows, group, dtype, zeros=False, scale_type=F16):
    codes, scales, z = q4_weights(seed, rows, cols, group, zeros, scale_type)
    x = torch.randn(tokens, cols, generator=gen(seed + 1)).to(dtype)
    want, size = q4(x, codes, scales, z)
    y = dense.q4_product(x.cuda(), codes.cuda(), scales.cuda(), None if z is None else z.cuda())
    near(y, want, tolerance(want, size, dtype, cols, group), "y")


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
def test_types_and_groups(dtype, group, zeros):
    compare(1, 3, 640, 50, group, dtype, zeros)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("tokens", [1, 2, 5, 6, 8, 10, 11, 16, 17, 21, 22, 32, 33, 64, 65, 130])
def test_tokens(tokens, dtype):
    compare(2, tokens, 512, 40, 128, dtype, True)


@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 63, 64, 65, 257, 1000])
@pytest.mark.parametrize("tokens", [1, 40])
def test_rows(rows, tokens):
    compare(3, tokens, 256, rows, 64, BF16)


@pytest.mark.parametrize("cols,group", [(32, 32), (64, 64), (64, 32), (96, 32), (128, 128), (160, 32), (192, 64),
                                        (224, 32), (384, 128), (1056, 32), (2592, 32), (4096, 128), (8256, 64)])
@pytest.mark.parametrize("tokens,dtype", [(1, BF16), (3, F32), (70, F16)])
def test_columns(cols, group, tokens, dtype):
    compare(4, tokens, cols, 33, group, dtype, True)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("tokens,rows", [(128, 512), (200, 1030), (512, 257), (300, 2048)])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_chunks(tokens, rows, group, dtype):
    """Prefill chunks of many tiles each way."""
    compare(5, tokens, 384, rows, group, dtype, group == 64)


# Products large enough for tiles of 64 tokens: 64, 128 and 256 rows wide.
TILED = [(200, 1856, 4096), (70, 1184, 16400), (260, 640, 16500)]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("tokens,cols,rows,group,zeros", [(*TILED[0], 64, True), (*TILED[0], 32, False),
                                                          (*TILED[1], 32, True), (*TILED[1], 32, False),
                                                          (*TILED[2], 128, False), (*TILED[2], 128, True),
                                                          (*TILED[2], 64, False)])
def test_tiles(tokens, cols, rows, group, zeros, dtype):
    compare(15, tokens, cols, rows, group, dtype, zeros, BF16 if group == 64 else F16)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_tiles_views_and_bad_tokens(dtype):
    """x and y at odd elements of wider rows; a token with an infinity or NaN
    has no finite output and the others keep their bits; zeros and magnitudes
    far from one in rows of their own."""
    codes, scales, z = q4_weights(16, 8200, 1536, 128, True)
    x = torch.randn(130, 1536, generator=gen(17))
    x[5], x[6], x[7] = 0.0, x[6] * (2e3 if dtype == F16 else 1e30), x[7] * (2e-3 if dtype == F16 else 1e-30)
    x[8] *= torch.logspace(-4, 3, 1536)
    x = x.to(dtype)
    want, size = q4(x, codes, scales, z)
    wide = torch.full((130, 1541), float("nan"), dtype=dtype).cuda()
    wide[:, 3:1539] = x.cuda()
    out = torch.full((130, 8207), 4.0, dtype=dtype).cuda()
    dev = [t.cuda() for t in (codes, scales, z)]
    y = dense.q4_product(wide[:, 3:1539], *dev, out=out[:, 5:8205])
    near(y, want, tolerance(want, size, dtype, 1536, 128) + (1e-36 if dtype != F16 else 2.0 ** -25), "y")
    assert (out[:, :5] == 4.0).all() and (out[:, 8205:] == 4.0).all()
    clean = y.clone()
    wide[0, 80], wide[129, 700] = float("inf"), float("nan")
    dense.q4_product(wide[:, 3:1539], *dev, out=out[:, 5:8205])
    assert torch.equal(y[1:129], clean[1:129]) and not torch.isfinite(y[::129]).any()


def test_tiles_in_a_graph():
    codes, scales, _ = (t.cuda() if t is not None else None for t in q4_weights(18, 8200, 1536, 128, False))
    x = torch.randn(130, 1536, generator=gen(19)).to(BF16).cuda()
    keep = x.clone()
    dense.q4_product(x, codes, scales)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = dense.q4_product(x, codes, scales)
    for k in (1.0, -2.0, 0.5):
        x.copy_(keep * k)
        y.fill_(1.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, dense.q4_product(x, codes, scales))
        torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("tokens", [2, 150])
def test_bf16_scales(dtype, tokens):
    compare(6, tokens, 256, 96, 32, dtype, True, BF16)


@pytest.mark.parametrize("tokens", [4, 150])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_views(tokens, dtype):
    """x and y within wider rows, at odd elements; nothing beside y is written."""
    codes, scales, _ = q4_weights(7, 300, 256, 64, False)
    x = torch.randn(tokens, 256, generator=gen(8)).to(dtype)
    want, size = q4(x, codes, scales, None)
    wide = torch.full((tokens, 261), float("nan"), dtype=dtype).cuda()
    wide[:, 3:259] = x.cuda()
    out = torch.full((tokens, 307), 4.0, dtype=dtype).cuda()
    dense.q4_product(wide[:, 3:259], codes.cuda(), scales.cuda(), out=out[:, 5:305])
    near(out[:, 5:305], want, tolerance(want, size, dtype, 256, 64), "y")
    assert (out[:, :5] == 4.0).all() and (out[:, 305:] == 4.0).all()


@pytest.mark.parametrize("tokens", [2, 150])
def test_extremes(tokens):
    """Magnitudes from 1e-30 to 1e30 in one call, and all codes at either end."""
    codes, scales, z = q4_weights(9, 70, 256, 64, True)
    codes[:10], codes[10:20] = 0, 255
    x = torch.randn(tokens, 256, generator=gen(10)) * torch.logspace(-30, 30, tokens)[:, None]
    want, size = q4(x, codes, scales, z)
    y = dense.q4_product(x.cuda(), codes.cuda(), scales.cuda(), z.cuda())
    near(y, want, tolerance(want, size, F32, 256, 64) + 1e-36, "y")


@pytest.mark.parametrize("tokens", [3, 150])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_a_bad_token_stays_its_own(tokens, dtype):
    """A token with an infinity or NaN has no finite output; the others keep
    their bits."""
    codes, scales, z = (t.cuda() for t in q4_weights(11, 100, 512, 128, True))
    x = torch.randn(tokens, 512, generator=gen(12)).to(dtype).cuda()
    clean = dense.q4_product(x, codes, scales, z)
    x[0, 77], x[2, 300] = float("inf"), float("nan")
    y = dense.q4_product(x, codes, scales, z)
    ok = torch.ones(tokens, dtype=torch.bool)
    ok[0] = ok[2] = False
    assert torch.equal(y[ok], clean[ok]) and not torch.isfinite(y[~ok]).any()


@pytest.mark.parametrize("tokens", [1, 7, 200])
def test_repeat_stream_and_graph(tokens):
    codes, scales, z = (t.cuda() for t in q4_weights(13, 520, 1024, 128, True))
    x = torch.randn(tokens, 1024, generator=gen(14)).to(BF16).cuda()
    want = dense.q4_product(x, codes, scales, z)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = dense.q4_product(x, codes, scales, z)
    s.synchronize()
    assert torch.equal(y, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = dense.q4_product(x, codes, scales, z)
    keep = x.clone()
    for k in (1.0, -2.0, 0.5):
        x.copy_(keep * k)
        y.fill_(1.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, dense.q4_product(x, codes, scales, z))
        torch.cuda.synchronize()


def test_nothing_to_do_and_refusals():
    codes, scales, z = (t.cuda() for t in q4_weights(15, 8, 128, 64, True))
    x = torch.ones(2, 128, dtype=BF16, device="cuda")
    assert dense.q4_product(x[:0], codes, scales, z).shape == (0, 8)
    assert dense.q4_product(x, codes[:0], scales[:0]).shape == (2, 0)
    for bad in (dict(x=x.double()), dict(x=x[0]), dict(codes=codes[:, :32]), dict(codes=codes.int()),
                dict(scales=scales.float()), dict(scales=scales[:, :1], zeros=None, codes=codes[:, :48].contiguous()),
                dict(zeros=z[:4]), dict(zeros=z.int()), dict(codes=codes.t()), dict(x=x.t()),
                dict(out=torch.empty(2, 9, dtype=BF16, device="cuda")), dict(x=torch.ones(4097, 128, dtype=BF16, device="cuda"))):
        with pytest.raises(ValueError):
            dense.q4_product(**{**dict(x=x, codes=codes, scales=scales, zeros=z), **bad})
