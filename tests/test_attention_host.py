"""Positions, prompt attention, draft trees and moves within the cache without a
GPU: what the calls refuse and in which order, the workspaces they ask for, and
the frequencies of scaled positions."""
import ctypes as C
import math

import pytest
import torch

import fronk_amd as fa
from fronk_amd import dense
from test_dense_host import CACHE_REFUSALS, P, cache_request, no_engine


def rotary_request(**kw):
    d = dict(tokens=3, heads=4, kv_heads=2, dim=128, pairs=32, type=dense.BF16, flags=0, magnitude=1.0, q=P, k=P, q_out=P,
             k_out=P, q_token=512, q_head=128, k_token=256, k_head=128, qo_token=512, qo_head=128, ko_token=256,
             ko_head=128, positions=P, frequencies=P)
    d.update(kw)
    return dense.RotaryRequest(**d)


def prompt_request(**kw):
    d = dict(sequences=2, tokens=10, k_tokens=20, max_tokens=8, max_context=16, heads=4, kv_heads=2, dim=128,
             type=dense.BF16, scale=1.0, q=P, k=P, v=P, o=P, q_token=512, q_head=128, k_token=256, k_head=128, v_token=256,
             v_head=128, o_token=512, o_head=128, offsets=P, k_offsets=P, status=None)
    d.update(kw)
    return dense.PromptRequest(**d)


def tree_request(cache=None, **kw):
    d = dict(sequences=2, tokens=10, max_tokens=8, heads=8, max_context=100, type=dense.BF16, table_stride=4, scale=1.0,
             q=P, o=P, q_token=1024, q_head=128, o_token=1024, o_head=128, tree=P, offsets=P, table=P, length=P, status=None)
    d.update(kw)
    return dense.TreeRequest(cache=cache or cache_request(), **d)


def moves_request(cache=None, **kw):
    d = dict(groups=2, moves=3, source=P, target=P, status=None)
    d.update(kw)
    return dense.MovesRequest(cache=cache or cache_request(), **d)


def copies_request(cache=None, **kw):
    d = dict(count=3, source=P, target=P, status=None)
    d.update(kw)
    return dense.CopiesRequest(cache=cache or cache_request(), **d)


NAN = float("nan")


@pytest.mark.parametrize("change,rc", [
    (dict(type=3), fa.INVALID), (dict(flags=2), fa.INVALID), (dict(dim=0), fa.INVALID), (dict(pairs=0), fa.INVALID),
    (dict(pairs=65), fa.INVALID), (dict(magnitude=NAN), fa.INVALID), (dict(tokens=1 << 31), fa.INVALID),
    (dict(q=None), fa.INVALID), (dict(k=None), fa.INVALID), (dict(q_out=None), fa.INVALID), (dict(k_out=None), fa.INVALID),
    (dict(positions=None), fa.INVALID), (dict(frequencies=None), fa.INVALID), (dict(frequencies=P + 4), fa.INVALID),
    (dict(positions=P + 2), fa.INVALID), (dict(q=P + 1), fa.INVALID), (dict(qo_token=1024), fa.INVALID),
    (dict(ko_head=256), fa.INVALID), (dict(dim=1026), fa.UNSUPPORTED), (dict(heads=65536), fa.UNSUPPORTED),
    (dict(kv_heads=65536), fa.UNSUPPORTED), (dict(tokens=(1 << 31) - 1, pairs=1, dim=4), fa.UNSUPPORTED),
    (dict(), fa.STATE), (dict(tokens=0, positions=None, q=None), fa.STATE), (dict(k=None, k_out=None, kv_heads=0), fa.STATE),
    (dict(q=None, q_out=None, heads=0), fa.STATE), (dict(q_out=2 * P, qo_token=640), fa.STATE), (dict(dim=1024, pairs=512), fa.STATE)])
def test_rotary_refusals(change, rc):
    no_engine()
    r = rotary_request(**change)
    assert fa.lib().fr_hip_rotate(C.addressof(r), None) == rc


@pytest.mark.parametrize("change,rc", [
    (dict(type=3), fa.INVALID), (dict(heads=0), fa.INVALID), (dict(kv_heads=0), fa.INVALID), (dict(heads=5), fa.INVALID),
    (dict(dim=0), fa.INVALID), (dict(scale=NAN), fa.INVALID), (dict(scale=float("inf")), fa.INVALID),
    (dict(tokens=1 << 31), fa.INVALID), (dict(k_tokens=(1 << 31) - 1), fa.INVALID), (dict(q=None), fa.INVALID),
    (dict(k=None), fa.INVALID), (dict(v=None), fa.INVALID), (dict(o=None), fa.INVALID), (dict(v=P + 1), fa.INVALID),
    (dict(o=P + 1), fa.INVALID), (dict(offsets=None), fa.INVALID), (dict(offsets=None, k_offsets=None, max_tokens=5), fa.INVALID),
    (dict(dim=96), fa.UNSUPPORTED), (dict(dim=512), fa.UNSUPPORTED), (dict(heads=130), fa.UNSUPPORTED),
    (dict(heads=1025, kv_heads=1025), fa.UNSUPPORTED), (dict(tokens=1 << 30), fa.UNSUPPORTED),
    (dict(sequences=1 << 24), fa.UNSUPPORTED), (dict(), None), (dict(tokens=0, q=None, o=None), None), (dict(sequences=0), None),
    (dict(k_tokens=0, k=None, v=None), None), (dict(offsets=None, max_tokens=5), None), (dict(k_offsets=None), None),
    (dict(offsets=None, k_offsets=None, max_tokens=5, max_context=10), None), (dict(max_tokens=1 << 31), None),
    (dict(max_context=0), None), (dict(max_context=1 << 31), None)])
def test_prompt_refusals(change, rc):
    """None: accepted, up to the engine that is not open."""
    no_engine()
    r, lib = prompt_request(**change), fa.lib()
    n = lib.fr_hip_prompt_workspace(C.addressof(r))
    assert lib.fr_hip_prompt_attend(C.addressof(r), P if n else None, n, None) == (fa.STATE if rc is None else rc)
    assert n == 0


@pytest.mark.parametrize("change,rc", [
    (dict(type=3), fa.INVALID), (dict(heads=0), fa.INVALID), (dict(heads=7), fa.INVALID), (dict(scale=NAN), fa.INVALID),
    (dict(tokens=1 << 31), fa.INVALID), (dict(q=None), fa.INVALID), (dict(o=None), fa.INVALID), (dict(tree=None), fa.INVALID),
    (dict(tree=P + 4), fa.INVALID), (dict(length=None), fa.INVALID), (dict(table=None), fa.INVALID), (dict(q=P + 1), fa.INVALID),
    (dict(offsets=None), fa.INVALID), (dict(table_stride=3), fa.INVALID),
    (dict(max_context=(1 << 31) - 1, table_stride=1 << 30), fa.INVALID), (dict(max_tokens=65), fa.UNSUPPORTED),
    (dict(heads=130), fa.UNSUPPORTED), (dict(sequences=1 << 24), fa.UNSUPPORTED), (dict(), None),
    (dict(max_context=0, table=None, table_stride=0), None), (dict(offsets=None, max_tokens=5), None),
    (dict(sequences=0, q=None, length=None), None), (dict(max_tokens=64), None), (dict(tokens=0, q=None), None)])
def test_tree_refusals(change, rc):
    no_engine()
    r, lib = tree_request(**change), fa.lib()
    n = lib.fr_hip_tree_workspace(C.addressof(r))
    assert lib.fr_hip_kv_attend_tree(C.addressof(r), P if n else None, n, None) == (fa.STATE if rc is None else rc)
    assert n == 0


@pytest.mark.parametrize("change,rc", CACHE_REFUSALS)
def test_cache_refusals(change, rc):
    no_engine()
    lib, c = fa.lib(), cache_request(**change)
    assert lib.fr_hip_kv_move(C.addressof(moves_request(c)), None) == rc
    assert lib.fr_hip_kv_copy(C.addressof(copies_request(c)), None) == rc
    if c.heads in (1, 2, 1025):
        r = tree_request(c, heads=max(2, c.heads), table_stride=1 << 23)
        assert lib.fr_hip_kv_attend_tree(C.addressof(r), None, 0, None) == rc
        assert lib.fr_hip_tree_workspace(C.addressof(r)) == 0


def test_trees_of_too_many_blocks_are_refused():
    """Places of 16 tokens and a head are numbered by 32 bits, the last number for none."""
    no_engine()
    lib = fa.lib()
    for pages, heads, rc in ((1 << 24, 64, fa.UNSUPPORTED), ((1 << 24) - 1, 64, fa.STATE)):
        r = tree_request(cache_request(pages=pages, heads=heads, page=64), heads=heads)
        assert lib.fr_hip_kv_attend_tree(C.addressof(r), None, 0, None) == rc
        assert lib.fr_hip_tree_workspace(C.addressof(r)) == 0


@pytest.mark.parametrize("change,rc", [
    (dict(source=None), fa.INVALID), (dict(target=None), fa.INVALID), (dict(groups=1 << 31, moves=1), fa.INVALID),
    (dict(moves=65), fa.UNSUPPORTED), (dict(groups=1 << 23, moves=1), fa.UNSUPPORTED), (dict(moves=64), fa.STATE),
    (dict(moves=0, source=None), fa.STATE), (dict(groups=0, source=None, target=None), fa.STATE)])
def test_move_refusals(change, rc):
    no_engine()
    r = moves_request(**change)
    assert fa.lib().fr_hip_kv_move(C.addressof(r), None) == rc


@pytest.mark.parametrize("change,rc", [
    (dict(source=None), fa.INVALID), (dict(target=None), fa.INVALID), (dict(count=1 << 31), fa.INVALID),
    (dict(count=1 << 24), fa.UNSUPPORTED), (dict(count=0, source=None, target=None), fa.STATE), (dict(), fa.STATE)])
def test_copy_refusals(change, rc):
    no_engine()
    r = copies_request(**change)
    assert fa.lib().fr_hip_kv_copy(C.addressof(r), None) == rc


def test_workspaces_are_checked_and_null_requests_are_refused():
    no_engine()
    lib = fa.lib()
    assert lib.fr_hip_rotate(None, None) == fa.INVALID
    assert lib.fr_hip_kv_move(None, None) == fa.INVALID and lib.fr_hip_kv_copy(None, None) == fa.INVALID
    few = prompt_request(sequences=1, tokens=16, max_tokens=16, k_tokens=65536, max_context=65536)
    tree = tree_request(cache_request(pages=4096), max_context=65536, table_stride=2048)
    for attend, size, r in ((lib.fr_hip_prompt_attend, lib.fr_hip_prompt_workspace, few),
                            (lib.fr_hip_kv_attend_tree, lib.fr_hip_tree_workspace, tree)):
        assert attend(None, None, 0, None) == fa.INVALID and size(None) == 0
        n = size(C.addressof(r))
        assert n > 0
        for w, given in ((None, n), (P, n - 1), (P + 8, n)):
            assert attend(C.addressof(r), w, given, None) == fa.INVALID
        assert attend(C.addressof(r), P, n, None) == fa.STATE


def test_python_checks_come_before_the_call():
    x, f = torch.zeros(2, 2, 64), torch.ones(4, dtype=torch.float64)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        dense.rotary(x, x, i, f)
    with pytest.raises(ValueError, match="GPU"):
        dense.prompt_attend(x, x, x)
    c = dense.KVCache.empty(2, 1, 16, 64, device="cpu")
    for call in (lambda: dense.kv_attend_tree(c, x, i.long(), i[:, None], i), lambda: dense.kv_move(c, i, i),
                 lambda: dense.kv_copy(c, i, i)):
        with pytest.raises(ValueError, match="uint8"):
            call()


def test_frequencies():
    f, m = dense.rotary_frequencies(8, 10000.0, device="cpu")
    assert m == 1.0 and f.dtype == torch.float64
    assert torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-15)
    g, m = dense.rotary_frequencies(8, factor=4.0, device="cpu")
    assert m == 1.0 and torch.equal(g, f / 4)
    # Turns in 2 pi 100 positions: 100, 10, 1, 0.1; kept from 20 on, divided up to 2.
    g, m = dense.rotary_frequencies(8, factor=4.0, context=200 * math.pi, slow=2.0, fast=20.0, device="cpu")
    kept = torch.tensor([1.0, 8 / 18, 0.0, 0.0], dtype=torch.float64)
    assert torch.allclose(g, f * (kept + (1 - kept) / 4), rtol=1e-14) and m == 1 + 0.1 * math.log(4)
    for bad in (dict(dim=0), dict(dim=7), dict(dim=8, factor=0.5), dict(dim=8, factor=NAN), dict(dim=8, factor=2.0, context=9, slow=3.0, fast=3.0)):
        with pytest.raises(ValueError):
            dense.rotary_frequencies(**bad, device="cpu")
