"""Outputs that share memory with an input are refused whatever the strides are, and those
that stand between an input's rows are not: the check itself, compiled for the host, against
all addresses, and the attention layer's operators over views of one projection's rows."""
import ctypes as C
import os
import random
import subprocess

import pytest

from test_attention_devices import BEGIN, folder, run   # noqa: F401 (a fixture)

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SHIM = r'''
#include "overlap.h"
typedef const int64_t* L;
extern "C" int share(int64_t at, int64_t e, int64_t n, L sizes, L strides, int64_t at2, int64_t e2, int64_t n2, L sizes2, L strides2) {
  return fronk::share({(uintptr_t)at, e, n, sizes, strides}, {(uintptr_t)at2, e2, n2, sizes2, strides2});
}
extern "C" int shares(int64_t at, int64_t e, int64_t n, L sizes, L strides) { return fronk::shares({(uintptr_t)at, e, n, sizes, strides}); }
'''


@pytest.fixture(scope="module")
def shim(tmp_path_factory):
    d = tmp_path_factory.mktemp("overlap")
    (d / "shim.cpp").write_text(SHIM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", "-fsanitize=undefined",
                    "-fno-sanitize-recover", "-shared", "-fPIC", "-I" + os.path.join(ROOT, "fronk_amd", "host"),
                    str(d / "shim.cpp"), "-o", str(d / "shim.so")], check=True)
    return C.CDLL(str(d / "shim.so"))


def longs(x):
    return (C.c_int64 * max(len(x), 1))(*x)


def share(shim, a, b):
    args = []
    for at, element, sizes, strides in (a, b):
        args += [C.c_int64(at), C.c_int64(element), C.c_int64(len(sizes)), longs(sizes), longs(strides)]
    return bool(shim.share(*args))


def shares(shim, at, element, sizes, strides):
    return bool(shim.shares(C.c_int64(at), C.c_int64(element), C.c_int64(len(sizes)), longs(sizes), longs(strides)))


def places(at, element, sizes, strides):
    out = [at]
    for n, s in zip(sizes, strides):
        out = [x + i * s * element for x in out for i in range(n)]
    return {x + e for x in out for e in range(element)}


def test_against_all_addresses(shim):
    r, seen = random.Random(1), [0, 0]
    for _ in range(6000):
        arrays = []
        for _ in range(2):
            n = r.randint(0, 3)
            strides = [r.choice([0, 1, 1, 2, 3, 4, 6, 7, 8, 12, 24, 25]) for _ in range(n)]
            arrays.append((r.randint(0, 160), r.choice([1, 2, 4, 8]), [r.randint(1, 5) for _ in range(n)], strides))
        want = bool(places(*arrays[0]) & places(*arrays[1]))
        seen[want] += 1
        assert share(shim, *arrays) == share(shim, *arrays[::-1]) == want, arrays
    assert min(seen) > 1000


def test_elements_of_one_array(shim):
    r, seen = random.Random(2), [0, 0]
    for _ in range(6000):
        n = r.randint(0, 4)
        strides = [r.choice([0, 1, 2, 3, 4, 5, 6, 8, 10, 12, 15, 20, 24, 40, 60, 120]) for _ in range(n)]
        a = (r.randint(0, 9), r.choice([1, 2, 4, 8]), [r.randint(1, 5) for _ in range(n)], strides)
        count = a[1]
        for x in a[2]:
            count *= x
        want = len(places(*a)) < count
        seen[want] += 1
        assert shares(shim, *a) == want, a
    assert min(seen) > 1000
    rows = lambda each, step: (1 << 40, 2, [100000, 20, 128], [each, step, 1])
    assert not shares(shim, *rows(24 * 128, 128)) and not shares(shim, *rows(128, 100000 * 128))
    assert shares(shim, *rows(19 * 128, 128)) and shares(shim, *rows(24 * 128, 127)) and shares(shim, *rows(128, 128))


def test_rows_of_one_projection(shim):
    """Heads a .. b of rows of `each` elements, of many tokens: two of them share memory where the heads do."""
    tokens, dim, heads = 100000, 128, 24
    each = heads * dim
    view = lambda a, b: (1 << 40 | a * dim * 2, 2, [tokens, b - a, dim], [each, dim, 1])
    for (a, b), (c, d) in [((0, 16), (16, 20)), ((0, 16), (15, 20)), ((20, 24), (0, 20)), ((0, 24), (23, 24)), ((3, 4), (4, 5))]:
        assert share(shim, view(a, b), view(c, d)) == (max(a, c) < min(b, d))
    # Every other head, every third value, another number of tokens.
    odd = lambda first, step: (1 << 40 | first * dim * 2, 2, [tokens - 5, heads // step, dim], [each, step * dim, 1])
    assert not share(shim, odd(0, 2), odd(1, 2)) and share(shim, odd(0, 2), odd(2, 4)) and not share(shim, odd(1, 2), odd(2, 4))
    assert share(shim, odd(0, 2), odd(1, 3))
    part = lambda first: (1 << 40 | first * 2, 2, [tokens, heads * dim // 3], [each, 3])
    assert not share(shim, part(0), part(1)) and share(shim, part(0), part(3))


OUTPUTS = """
{body}
def refused(f, args, why="out"):
    n = calls.value
    try:
        f(*args)
    except ValueError as e:
        assert why in str(e) and calls.value == n, str(e)
    else:
        raise AssertionError("was not refused")


def taken(f, args):
    n = calls.value
    f(*args)
    assert calls.value == n + 1


mode = FakeTensorMode()
with mode:
    rows = torch.empty(9, 8 * 64 + 16, dtype=torch.bfloat16, device="cuda:0")
    h = lambda a, b: rows[:, a * 64:b * 64].unflatten(1, (b - a, 64))
    three = torch.empty(9, dtype=torch.int32, device="cuda:0")
    f = torch.empty(32, dtype=torch.float64, device="cuda:0")
    fresh = torch.empty(9, 2, 64, dtype=torch.bfloat16, device="cuda:0")
    rotary = lambda q, k, out: [q, k, three, f, False, 1.0, out]
    prompt = lambda q, k, v, out: [q, k, v, None, None, None, None, None, out, None]
    R, P = _attention.rotary, _attention.prompt_attend
    q, k, v = h(0, 2), h(2, 4), h(4, 6)
    # In place, apart, and between the rows.
    for out in ((q, k), (fresh, k), (q, fresh), (h(4, 6), h(6, 8)), (h(6, 8), k), None):
        taken(R, rotary(q, k, out))
    taken(R, rotary(q, None, (q, None))), taken(R, rotary(q, None, (h(2, 4), None)))
    for out in ((h(1, 3), fresh), (h(1, 3), h(4, 6)), (h(2, 4), h(4, 6)), (h(4, 6), h(1, 3)), (h(4, 6), h(0, 2)), (h(4, 6), h(5, 7)),
                (k, q), (h(3, 5), k), (q, h(3, 5)), (rows[:, 64:192].unflatten(1, (2, 64)), fresh)):
        refused(R, rotary(q, k, out))
    for out in (fresh, h(6, 8), None):
        taken(P, prompt(q, k, v, out))
    for a in range(6):
        refused(P, prompt(q, k, v, h(a, a + 2)))
    refused(P, prompt(q[:8], k[1:], v[1:], rows[1:, 64:192].unflatten(1, (2, 64))))
"""


def test_views_of_a_projections_rows(folder):   # noqa: F811
    run(folder, OUTPUTS.replace("{body}", ""))


def test_outputs_whose_elements_share_memory(folder):   # noqa: F811
    run(folder, """
mode = FakeTensorMode()
with mode:
    b = torch.empty(4096, dtype=torch.bfloat16, device="cuda:0")
    x = lambda: torch.empty(9, 2, 64, dtype=torch.bfloat16, device="cuda:0")
    for strides in ((64, 64, 1), (127, 64, 1), (128, 63, 1), (0, 64, 1), (64, 128, 1)):
        try:
            _attention.prompt_attend(x(), x(), x(), None, None, None, None, None, b.as_strided((9, 2, 64), strides), None)
        except ValueError as e:
            assert "places of its own" in str(e), str(e)
        else:
            raise AssertionError(strides)
    assert calls.value == 0
    for strides in ((128, 64, 1), (64, 640, 1), (192, 64, 1), (129, 65, 1)):
        _attention.prompt_attend(x(), x(), x(), None, None, None, None, None, b.as_strided((9, 2, 64), strides), None)
    assert calls.value == 4
""")


WHOLE = """
mode = FakeTensorMode()


def each(name, make, call, names):
    # All inputs apart from out, then each in turn in its first bytes, and in its last.
    with mode:
        for victim in [None] + names:
            for end in (False, True):
                args = make()
                size = 4 * 9 * 2 * 64
                if victim is not None:
                    t = args[victim]
                    flat = torch.empty(2 * size + t.numel() * t.element_size(), dtype=torch.uint8, device="cuda:0")
                    at = 0 if end else size - t.element_size()
                    args[victim] = flat[at:at + t.numel() * t.element_size()].view(t.dtype).view(t.shape)
                    first = (t.numel() - 1) * t.element_size() // 8 * 8 if end else 0
                    out = flat[first:first + size].view(torch.float32).view(9, 2, 64)
                else:
                    out = torch.empty(9, 2, 64, device="cuda:0")
                n = calls.value
                try:
                    call(args, out)
                except ValueError as e:
                    assert victim is not None and "out shares memory" in str(e), (name, victim, end, str(e))
                else:
                    assert victim is None and calls.value == n + 1, (name, victim, end)


def t(*shape, dtype=torch.float32):
    return torch.empty(*shape, dtype=dtype, device="cuda:0")


i32, i64, u8 = torch.int32, torch.int64, torch.uint8
{cases}
"""


def test_outputs_over_what_is_looked_up(folder):   # noqa: F811
    """Offsets, tables, words and lengths count as inputs as q does: other workgroups, and the join of a context's
    stretches, read them when some outputs are written."""
    run(folder, WHOLE.replace("{cases}", """
each("prompt", lambda: dict(q=t(9, 2, 64), k=t(12, 1, 64), v=t(12, 1, 64), offsets=t(3, dtype=i32), k_offsets=t(3, dtype=i32)),
     lambda a, out: _attention.prompt_attend(a["q"], a["k"], a["v"], a["offsets"], a["k_offsets"], 9, 12, None, out, None),
     ["q", "k", "v", "offsets", "k_offsets"])
each("tree", lambda: dict(q=t(9, 2, 64), tree=t(9, dtype=i64), table=t(2, 3, dtype=i32), lengths=t(2, dtype=i32), offsets=t(3, dtype=i32),
                          k=t(2, 1, 16, 64, dtype=u8), v=t(2, 1, 1, 64, 16, dtype=u8), ke=t(2, 1, 16, dtype=u8), ve=t(2, 1, 16, dtype=u8)),
     lambda a, out: _attention.kv_attend_tree((a["k"], a["v"], a["ke"], a["ve"]), a["q"], a["tree"], a["table"], a["lengths"], a["offsets"],
                                              None, None, None, out, None),
     ["q", "tree", "table", "lengths", "offsets", "k", "v", "ke", "ve"])
"""))
