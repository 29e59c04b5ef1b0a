"""The dense operators without a GPU: what the calls refuse and in which order
(arguments before the engine's state), the workspaces they ask for, and the
bounds checks and cache addresses of the kernels, compiled for the host."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest
import torch

import fronk_amd as fa
from fronk_amd import dense

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 1 << 20   # an address that nothing follows here


def delta_request(**kw):
    d = dict(sequences=2, tokens=10, max_tokens=8, key_heads=2, heads=4, key_dim=128, value_dim=128, type=dense.BF16,
             flags=0, slots=2, scale=1.0, q=P, k=P, v=P, g=P, beta=P, o=P, q_token=256, q_head=128, k_token=256,
             k_head=128, v_token=512, v_head=128, o_token=512, o_head=128, g_token=4, beta_token=4, offsets=P,
             slot=None, state_in=P, state_out=P, status=None)
    d.update(kw)
    return dense.DeltaRequest(**d)


def q4_request(**kw):
    d = dict(tokens=1, rows=64, cols=256, group=64, type=dense.BF16, scale_type=dense.F16, x=P, codes=P, scales=P,
             zeros=None, y=P, x_token=256, y_token=64)
    d.update(kw)
    return dense.Q4Request(**d)


def cache_request(**kw):
    d = dict(pages=4, heads=2, page=32, dim=128, k_codes=P, v_codes=P, k_exp=P, v_exp=P)
    d.update(kw)
    return dense.CacheRequest(**d)


def tokens_request(cache=None, **kw):
    d = dict(tokens=3, type=dense.BF16, k=P, v=P, k_token=256, k_head=128, v_token=256, v_head=128, slot=P, status=None)
    d.update(kw)
    return dense.TokensRequest(cache=cache or cache_request(), **d)


def query_request(cache=None, **kw):
    d = dict(sequences=2, burst=2, heads=8, max_context=100, type=dense.BF16, table_stride=4, scale=1.0, q=P, o=P,
             q_token=1024, q_head=128, o_token=1024, o_head=128, table=P, length=P, status=None)
    d.update(kw)
    return dense.QueryRequest(cache=cache or cache_request(), **d)


def no_engine():
    lib = fa.lib()
    if lib.fr_hip_release(0) != fa.STATE:
        pytest.skip("another test holds the engine open")


@pytest.mark.parametrize("change,rc", [
    (dict(type=3), fa.INVALID), (dict(flags=2), fa.INVALID), (dict(key_heads=0), fa.INVALID),
    (dict(heads=0), fa.INVALID), (dict(key_heads=3), fa.INVALID), (dict(key_dim=0), fa.INVALID),
    (dict(value_dim=0), fa.INVALID), (dict(scale=float("nan")), fa.INVALID), (dict(scale=float("inf")), fa.INVALID),
    (dict(offsets=None), fa.INVALID), (dict(slots=1), fa.INVALID), (dict(q=None), fa.INVALID),
    (dict(k=None), fa.INVALID), (dict(v=None), fa.INVALID), (dict(g=None), fa.INVALID), (dict(beta=None), fa.INVALID),
    (dict(o=None), fa.INVALID), (dict(state_in=P + 8), fa.INVALID), (dict(state_out=P + 4), fa.INVALID),
    (dict(q=P + 1), fa.INVALID), (dict(tokens=1 << 31), fa.INVALID),
    (dict(key_dim=96), fa.UNSUPPORTED), (dict(key_dim=512), fa.UNSUPPORTED), (dict(value_dim=40), fa.UNSUPPORTED),
    (dict(value_dim=1040), fa.UNSUPPORTED), (dict(heads=65536), fa.UNSUPPORTED),
    (dict(sequences=1 << 30, slots=1 << 30), fa.UNSUPPORTED)])
def test_delta_refusals(change, rc):
    no_engine()
    r = delta_request(**change)
    assert fa.lib().fr_hip_delta_rule(C.addressof(r), None, 0, None) == rc
    assert fa.lib().fr_hip_delta_workspace(C.addressof(r)) == 0


@pytest.mark.parametrize("change,rc", [
    (dict(type=3), fa.INVALID), (dict(scale_type=dense.F32), fa.INVALID), (dict(group=16), fa.INVALID),
    (dict(group=96), fa.INVALID), (dict(cols=0), fa.INVALID), (dict(cols=96), fa.INVALID), (dict(x=None), fa.INVALID),
    (dict(codes=None), fa.INVALID), (dict(scales=None), fa.INVALID), (dict(y=None), fa.INVALID),
    (dict(codes=P + 8), fa.INVALID), (dict(scales=P + 1), fa.INVALID), (dict(y=P + 1), fa.INVALID),
    (dict(type=dense.F32, x=P + 2), fa.INVALID), (dict(tokens=4097), fa.UNSUPPORTED),
    (dict(cols=65536 + 64), fa.UNSUPPORTED), (dict(rows=(1 << 28) + 1), fa.UNSUPPORTED)])
def test_q4_refusals(change, rc):
    no_engine()
    r = q4_request(**change)
    assert fa.lib().fr_hip_q4_product(C.addressof(r), None, 0, None) == rc
    assert fa.lib().fr_hip_q4_workspace(C.addressof(r)) == 0


CACHE_REFUSALS = [
    (dict(pages=0), fa.INVALID), (dict(heads=0), fa.INVALID), (dict(page=0), fa.INVALID), (dict(dim=0), fa.INVALID),
    (dict(k_codes=None), fa.INVALID), (dict(v_codes=None), fa.INVALID), (dict(k_exp=None), fa.INVALID),
    (dict(v_exp=P + 1), fa.INVALID), (dict(k_codes=P + 8), fa.INVALID), (dict(dim=96), fa.UNSUPPORTED),
    (dict(page=24), fa.UNSUPPORTED), (dict(page=4112), fa.UNSUPPORTED), (dict(pages=1 << 27), fa.UNSUPPORTED),
    (dict(heads=1025), fa.UNSUPPORTED)]


@pytest.mark.parametrize("change,rc", CACHE_REFUSALS)
def test_cache_refusals(change, rc):
    no_engine()
    lib, c = fa.lib(), cache_request(**change)
    r = tokens_request(c)
    assert lib.fr_hip_kv_append(C.addressof(r), None) == rc
    assert lib.fr_hip_kv_read(C.addressof(r), None) == rc
    wide = dict(heads=1025, table_stride=1 << 23) if c.heads == 1025 else dict(table_stride=1 << 23)
    if c.heads in (1, 2, 1025):
        r = query_request(c, **wide)
        assert lib.fr_hip_kv_attend(C.addressof(r), None, 0, None) == rc
        assert lib.fr_hip_kv_workspace(C.addressof(r)) == 0


@pytest.mark.parametrize("change,rc", [
    (dict(type=3), fa.INVALID), (dict(k=None), fa.INVALID), (dict(v=None), fa.INVALID), (dict(slot=None), fa.INVALID),
    (dict(k=P + 1), fa.INVALID), (dict(tokens=1 << 31), fa.INVALID), (dict(tokens=(1 << 31) - 1), fa.UNSUPPORTED)])
def test_append_refusals(change, rc):
    no_engine()
    r = tokens_request(cache_request(heads=1024, pages=1), **change)
    assert fa.lib().fr_hip_kv_append(C.addressof(r), None) == rc


@pytest.mark.parametrize("change,rc", [
    (dict(type=3), fa.INVALID), (dict(burst=0), fa.INVALID), (dict(heads=0), fa.INVALID), (dict(heads=7), fa.INVALID),
    (dict(scale=float("inf")), fa.INVALID), (dict(q=None), fa.INVALID), (dict(o=None), fa.INVALID),
    (dict(length=None), fa.INVALID), (dict(table=None), fa.INVALID), (dict(q=P + 1), fa.INVALID),
    (dict(table_stride=3), fa.INVALID), (dict(max_context=(1 << 31) - 1, table_stride=1 << 30), fa.INVALID),
    (dict(burst=9), fa.UNSUPPORTED), (dict(heads=130), fa.UNSUPPORTED),
    (dict(sequences=1 << 20), fa.UNSUPPORTED)])
def test_attend_refusals(change, rc):
    no_engine()
    r = query_request(**change)
    assert fa.lib().fr_hip_kv_attend(C.addressof(r), P, 1 << 40, None) == rc
    assert fa.lib().fr_hip_kv_workspace(C.addressof(r)) == 0


def test_workspace_is_checked_and_null_requests_are_refused():
    no_engine()
    lib = fa.lib()
    for fn in (lib.fr_hip_delta_rule, lib.fr_hip_q4_product, lib.fr_hip_kv_attend):
        assert fn(None, None, 0, None) == fa.INVALID
    assert lib.fr_hip_kv_append(None, None) == fa.INVALID and lib.fr_hip_kv_read(None, None) == fa.INVALID
    r = query_request(cache_request(pages=4096), max_context=4096, table_stride=128)
    n = lib.fr_hip_kv_workspace(C.addressof(r))
    assert n > 0
    for w, size in ((None, n), (P, n - 1), (P + 8, n)):
        assert lib.fr_hip_kv_attend(C.addressof(r), w, size, None) == fa.INVALID
    assert lib.fr_hip_kv_attend(C.addressof(r), P, n, None) == fa.STATE
    # Whole arguments and no engine: its state is what is reported.
    for fn, r in ((lib.fr_hip_kv_append, tokens_request()), (lib.fr_hip_kv_read, tokens_request(k=None))):
        assert fn(C.addressof(r), None) == fa.STATE
    r = q4_request()
    assert lib.fr_hip_q4_product(C.addressof(r), P, lib.fr_hip_q4_workspace(C.addressof(r)), None) == fa.STATE
    r = delta_request()
    assert lib.fr_hip_delta_rule(C.addressof(r), P, lib.fr_hip_delta_workspace(C.addressof(r)), None) == fa.STATE


def test_python_checks_come_before_the_call():
    x = torch.zeros(2, 128)
    with pytest.raises(ValueError, match="GPU"):
        dense.q4_product(x, torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.float16))
    with pytest.raises(ValueError, match="GPU"):
        dense.delta_rule(x[None], x[None], x[None], x, x)
    with pytest.raises(ValueError, match="uint8"):
        c = dense.KVCache.empty(2, 1, 16, 64, device="cpu")
        dense.kv_read(c, torch.zeros(1, dtype=torch.int32))


# ------------------------------------------------- the kernels' bounds checks

SHIM = r'''
#include "bounds.h"
extern "C" int locate(int32_t s, uint32_t n, uint32_t pages, uint32_t* out) { return fronk::locate(s, n, pages, out, out + 1); }
extern "C" int there(int32_t p, uint32_t pages) { return fronk::page_there(p, pages); }
extern "C" uint64_t exp_at(uint32_t h, uint32_t n, uint32_t p, uint32_t i, uint32_t a) { return fronk::exp_at(h, n, p, i, a); }
extern "C" uint64_t v_at(uint32_t h, uint32_t n, uint32_t d, uint32_t p, uint32_t i, uint32_t a) { return fronk::v_at(h, n, d, p, i, a); }
extern "C" uint32_t first_bytes(int n) { return fronk::first_bytes(n); }
extern "C" uint32_t bad(int32_t s, uint32_t n, int32_t a, int32_t b, uint32_t t, uint32_t m) { return fronk::bad_sequence(s, n, a, b, t, m); }
'''


@pytest.fixture(scope="module")
def shim(tmp_path_factory):
    d = tmp_path_factory.mktemp("bounds")
    (d / "shim.cpp").write_text(SHIM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", "-fsanitize=undefined",
                    "-fno-sanitize-recover", "-shared", "-fPIC", "-I" + os.path.join(ROOT, "fronk_amd", "csrc"),
                    str(d / "shim.cpp"), "-o", str(d / "shim.so")], check=True)
    L = C.CDLL(str(d / "shim.so"))
    L.exp_at.restype = L.v_at.restype = C.c_uint64
    L.first_bytes.restype = L.bad.restype = C.c_uint32
    return L


def test_slots_and_pages(shim):
    out = (C.c_uint32 * 2)()
    page, pages = 48, 5
    assert shim.locate(-1, page, pages, out) == 0
    for s in (0, 1, 47, 48, 239):
        assert shim.locate(s, page, pages, out) == 1 and tuple(out) == divmod(s, page)
    for s in (240, 241, -2, -48, 2 ** 31 - 1, -2 ** 31):
        assert shim.locate(s, page, pages, out) == 2
    assert [shim.there(p, pages) for p in (-2 ** 31, -1, 0, 4, 5, 2 ** 31 - 1)] == [0, 0, 1, 1, 0, 0]


def test_addresses_are_the_layouts(shim):
    pages, heads, page, dim = 3, 2, 32, 64
    k = np.arange(pages * heads * page).reshape(pages, heads, page)
    v = np.arange(pages * heads * page * dim).reshape(pages, heads, page // 16, dim, 16)
    for p in range(pages):
        for h in range(heads):
            for at in range(page):
                assert shim.exp_at(heads, page, p, h, at) == k[p, h, at]
                base = shim.v_at(heads, page, dim, p, h, at)
                for d in (0, 1, dim - 1):
                    assert base + 16 * d == v[p, h, at // 16, d, at % 16]
    # Past 32 bits.
    assert shim.exp_at(8, 4096, 500000, 7, 4095) == (500000 * 8 + 7) * 4096 + 4095
    assert shim.v_at(8, 4096, 256, 500000, 7, 17) == ((500000 * 8 + 7) * 4096 + 16) * 256 + 1


def test_tail_masks(shim):
    assert [shim.first_bytes(n) for n in (-5, 0, 1, 2, 3, 4, 5)] == \
        [0, 0, 0xff, 0xffff, 0xffffff, 0xffffffff, 0xffffffff]


def test_sequences(shim):
    ok = (3, 4, 10, 20, 20, 10)
    assert shim.bad(*ok) == 0 and shim.bad(-1, 4, 10, 20, 20, 10) == 0 and shim.bad(0, 1, 5, 5, 5, 0) == 0
    for s in (-2, 4, 2 ** 31 - 1, -2 ** 31):
        assert shim.bad(s, *ok[1:]) == dense.BAD_SLOT
    for a, b in ((-1, 5), (5, 4), (10, 21), (9, 20), (-2 ** 31, 2 ** 31 - 1), (0, -1)):
        assert shim.bad(3, 4, a, b, 20, 10) == dense.BAD_OFFSET
    assert shim.bad(9, 4, 5, 4, 20, 10) == dense.BAD_SLOT | dense.BAD_OFFSET


@pytest.mark.parametrize("change,rc", [
    # 4 heads of 128 columns: 32 workgroups a sequence, of 512 threads in chunks.
    (dict(sequences=1 << 18, tokens=1 << 18, slots=1 << 18, max_tokens=64), fa.UNSUPPORTED),
    (dict(sequences=(1 << 18) - 1, tokens=1 << 18, slots=1 << 18, max_tokens=64), None),
    (dict(sequences=1 << 20, tokens=1 << 20, slots=1 << 20, max_tokens=8), fa.UNSUPPORTED),
    (dict(sequences=(1 << 20) - 1, tokens=1 << 20, slots=1 << 20, max_tokens=8), None)])
def test_delta_grids_end_below_2_32_threads(change, rc):
    """None: accepted, up to the engine that is not open."""
    no_engine()
    r = delta_request(**change)
    n = fa.lib().fr_hip_delta_workspace(C.addressof(r))
    assert fa.lib().fr_hip_delta_rule(C.addressof(r), P if n else None, n, None) == (fa.STATE if rc is None else rc)


@pytest.mark.parametrize("tokens,rows,rc", [(4096, 1 << 24, fa.UNSUPPORTED), (4096, 1 << 23, None), (64, 1 << 28, None)])
def test_q4_grids_end_below_2_32_threads(tokens, rows, rc):
    no_engine()
    r = q4_request(tokens=tokens, rows=rows)
    n = fa.lib().fr_hip_q4_workspace(C.addressof(r))
    assert fa.lib().fr_hip_q4_product(C.addressof(r), P if n else None, n, None) == (fa.STATE if rc is None else rc)


def test_delta_workspace_for_the_order_of_many_sequences():
    """Above 2048 sequences, four bytes of each beside what chunks take."""
    no_engine()

    def size(**kw):
        r = delta_request(**kw)
        return fa.lib().fr_hip_delta_workspace(C.addressof(r))

    n = dict(tokens=5000, sequences=2048, slots=5000)
    more = {**n, "sequences": 2049}
    assert size(**n) == 0 and size(**more) == 4 * 2049
    assert size(sequences=2049, tokens=2049, slots=2049, offsets=None, max_tokens=1) == 0
    a, b = size(**n, max_tokens=64), size(**more, max_tokens=64)
    assert a > 0 and a % 1024 == 0 and b % 1024 == (4 * 2049) % 1024
    r = delta_request(**more)
    for w, given in ((None, 4 * 2049), (P, 4 * 2049 - 1), (P + 8, 4 * 2049)):
        assert fa.lib().fr_hip_delta_rule(C.addressof(r), w, given, None) == fa.INVALID
    assert fa.lib().fr_hip_delta_rule(C.addressof(r), P, 4 * 2049, None) == fa.STATE


def test_delta_goes_by_the_tokens_there_are():
    """A generous max_tokens is no reason for chunks, nor their workspace."""
    no_engine()
    for tokens, most, chunks in ((10, 4096, False), (32, 33, False), (33, 32, False), (33, 33, True), (0, 64, False)):
        r = delta_request(tokens=tokens, max_tokens=most)
        assert (fa.lib().fr_hip_delta_workspace(C.addressof(r)) > 0) == chunks, (tokens, most)


@pytest.mark.parametrize("rows,refused", [(-3, False), (-2, False), (-1, True), (0, False), (1, True), (2, False), (3, False)])
def test_delta_pools_are_one_or_apart(rows, refused):
    """Two rows each, `rows` rows from one to the other."""
    no_engine()
    r = delta_request(state_in=P * 64, state_out=P * 64 + rows * 4 * 128 * 128 * 4)
    assert fa.lib().fr_hip_delta_rule(C.addressof(r), None, 0, None) == (fa.INVALID if refused else fa.STATE)
    if rows:
        r = delta_request(state_in=P * 64, state_out=P * 64 + rows * 4 * 128 * 128 * 4 + (-16 if rows > 0 else 16))
        assert fa.lib().fr_hip_delta_rule(C.addressof(r), None, 0, None) == (fa.INVALID if abs(rows) < 3 else fa.STATE)


def test_attention_over_nothing_needs_no_table():
    no_engine()
    r = query_request(max_context=0, table=None, table_stride=0)
    assert fa.lib().fr_hip_kv_attend(C.addressof(r), None, 0, None) == fa.STATE
    r = query_request(max_context=1, table=None)
    assert fa.lib().fr_hip_kv_attend(C.addressof(r), None, 0, None) == fa.INVALID
