"""The example's layers, every operator of a pass against 64 bits on the operands
that it got, and its decoding from a graph against the same pass run eagerly."""
import importlib.util
import os

import pytest
import torch

from dense_fixtures import HALF, U, attend, delta, delta_tolerance, gen, near, q4
from fronk_amd import dense

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SMALL = dict(hidden=256, key_heads=2, heads=4, key_dim=64, value_dim=48, q_heads=6, kv_heads=2, dim=64, streams=3,
             context=160, page=32)


def example():
    spec = importlib.util.spec_from_file_location("dense_layers", os.path.join(ROOT, "examples", "dense_layers.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def close(got, x, weights, dtype, what):
    """A product of 4-bit weights: one rounding, and the fp32 sums' own."""
    codes, scales, zeros = (t.cpu() for t in weights)
    want, size = q4(x.cpu(), codes, scales, zeros)
    cols, group = x.shape[1], x.shape[1] // scales.shape[1]
    near(got, want, HALF[dtype] * want.abs() + (4 * (cols // 32) + 2 * (cols // group) + 16) * U * size, what)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_operators_of_a_pass(dtype):
    m = example()
    layers = m.Layers(**SMALL, dtype=dtype)
    key_heads, heads, dk, dv, q_heads, kv_heads, dim = layers.sizes
    done = [0, 0, 0]
    # Prompts of unequal length, one of them over two chunks, then a token each.
    for step, lens in enumerate([[70, 5, 1], [1, 1, 1], [1, 1, 1]]):
        x = torch.randn(sum(lens), 256, generator=gen(step)).to(dtype).cuda()
        position = torch.cat([torch.arange(n) + d for n, d in zip(lens, done)]).cuda()
        offsets = torch.tensor([0, lens[0], lens[0] + lens[1], sum(lens)], dtype=torch.int32).cuda()
        stream = torch.tensor([2, 0, 1], dtype=torch.int32).cuda()
        of = stream.long().cpu().repeat_interleave(torch.tensor(lens)).cuda()
        t = {}
        y = layers.forward(x, of, position, stream, offsets, max(lens), t)
        done = [d + n for d, n in zip(done, lens)]
        assert layers.status.item() == 0
        close(t["row"], x, layers.in1, dtype, "the first layer's projection")
        order = stream.long().cpu()
        want, final = delta(*(t[n].cpu() for n in ("q", "k", "v", "g", "beta")), t["before"].cpu()[order], lens,
                            dk ** -0.5, True)
        size = max(float(final.abs().max()), 1.0)
        near(t["o"], want, delta_tolerance(want, dtype, dk, max(lens), size), "the delta rule")
        near(layers.states.cpu()[order], final, delta_tolerance(final, torch.float32, dk, max(lens), size), "states")
        close(t["row2"], t["h"], layers.in2, dtype, "the second layer's projection")
        ks, vs = [], []
        for i in order:
            slots = layers.slots(i.cuda(), torch.arange(done[list(order).index(i)]).cuda())
            k, v = dense.kv_read(layers.cache, slots, torch.float32)
            ks.append(k.cpu()), vs.append(v.cpu())
        rows = torch.repeat_interleave(torch.arange(3), torch.tensor(lens))
        lengths = (position.cpu() + 1).tolist()
        want = attend(t["q2"].cpu(), [ks[i] for i in rows], [vs[i] for i in rows], lengths, 1, dim ** -0.5)
        top = max(float(v.abs().max()) for v in vs)
        scores = dim ** -0.5 * float(t["q2"].abs().max()) * max(float(k.abs().max()) for k in ks) * dim
        near(t["a"], want, HALF[dtype] * want.abs()
             + ((16 * scores + 64) * U + (0 if dtype == torch.float32 else 2.0 ** -17)) * top, "attention")
        assert torch.isfinite(y).all()


def test_decoding_from_a_graph():
    """Every replay gives the bits of the same pass run eagerly."""
    m = example()
    a, b = m.Layers(**SMALL, seed=3), m.Layers(**SMALL, seed=3)
    x = torch.randn(3 * 20, 256, generator=gen(9)).to(torch.bfloat16).cuda()
    stream, one = torch.arange(3, dtype=torch.int32).cuda(), torch.arange(3).cuda()
    position = torch.arange(20).repeat(3).cuda()
    offsets = torch.arange(4, dtype=torch.int32).cuda() * 20
    of = torch.arange(3).repeat_interleave(20).cuda()
    y = [layers.forward(x, of, position, stream, offsets, 20) for layers in (a, b)]
    assert torch.equal(*y)
    decoder = m.Decoder(a, 20)
    token = y[1].view(3, 20, 256)[:, -1]
    single = torch.arange(4, dtype=torch.int32).cuda()
    for n in range(4):
        decoder.x.copy_(token)
        decoder.graph.replay()
        torch.cuda.synchronize()
        token = b.forward(token, one, torch.full((3,), 20 + n).cuda(), stream, single, 1)
        assert torch.equal(decoder.y, token) and torch.equal(a.states, b.states)
        torch.cuda.synchronize()
    assert a.status.item() == 0
