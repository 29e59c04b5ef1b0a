"""The dense operators over torch tensors: thin calls of the C ABI
(include/fronk_hip.h), enqueued on torch's current stream, no compute and no
fallback of their own. Tensors are on the open engine's device (fr_hip_open;
the first call here opens the current device) and may have any strides but for
a contiguous last axis.

  delta_rule   the gated delta rule, decode bursts to prompts
  q4_product   products with 4-bit weights and group scales
  KVCache, kv_append, kv_read, kv_attend   the paged 8-bit key/value cache

A refused call raises ValueError before anything is enqueued. What only the
device can see (offsets, slots, pages, lengths) is bounds-checked there: a bad
entry reads and writes nothing and sets its bit (BAD_*) in `status`, an int32
tensor of one element that the caller clears.
"""
import ctypes as C
from typing import NamedTuple

import torch

from . import INVALID, OK, STATE, UNSUPPORTED, Engine, lib

F32, F16, BF16 = 0, 1, 2
BAD_OFFSET, BAD_SLOT, BAD_PAGE, BAD_LENGTH = 1, 2, 4, 8
DELTA_NORMALIZE = 1
# Of a stream argument: HIP's default stream (NULL is the library's own).
STREAM_DEFAULT = 1

_TYPES = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}
_u, _i64, _p, _f = C.c_uint, C.c_int64, C.c_void_p, C.c_float


class DeltaRequest(C.Structure):
    _fields_ = [(n, _u) for n in ("sequences", "tokens", "max_tokens", "key_heads", "heads", "key_dim", "value_dim",
                                  "type", "flags", "slots")] + [("scale", _f)] + \
        [(n, _p) for n in ("q", "k", "v", "g", "beta", "o")] + \
        [(n, _i64) for n in ("q_token", "q_head", "k_token", "k_head", "v_token", "v_head", "o_token", "o_head",
                             "g_token", "beta_token")] + \
        [(n, _p) for n in ("offsets", "slot", "state_in", "state_out", "status")]


class Q4Request(C.Structure):
    _fields_ = [(n, _u) for n in ("tokens", "rows", "cols", "group", "type", "scale_type")] + \
        [(n, _p) for n in ("x", "codes", "scales", "zeros", "y")] + [("x_token", _i64), ("y_token", _i64)]


class CacheRequest(C.Structure):
    _fields_ = [(n, _u) for n in ("pages", "heads", "page", "dim")] + \
        [(n, _p) for n in ("k_codes", "v_codes", "k_exp", "v_exp")]


class TokensRequest(C.Structure):
    """fr_hip_kv_write and fr_hip_kv_values."""
    _fields_ = [("cache", CacheRequest), ("tokens", _u), ("type", _u), ("k", _p), ("v", _p)] + \
        [(n, _i64) for n in ("k_token", "k_head", "v_token", "v_head")] + [("slot", _p), ("status", _p)]


class QueryRequest(C.Structure):
    _fields_ = [("cache", CacheRequest)] + \
        [(n, _u) for n in ("sequences", "burst", "heads", "max_context", "type", "table_stride")] + \
        [("scale", _f), ("q", _p), ("o", _p)] + \
        [(n, _i64) for n in ("q_token", "q_head", "o_token", "o_head")] + \
        [(n, _p) for n in ("table", "length", "status")]


_REASON = {INVALID: "invalid arguments", UNSUPPORTED: "sizes outside the supported range",
           STATE: "no open engine on this device"}


def _raise(rc, what):
    if rc in (INVALID, UNSUPPORTED):
        raise ValueError(f"{what}: {_REASON[rc]} ({rc})")
    raise RuntimeError(f"{what} failed with {rc} ({_REASON.get(rc, 'the device reported an error')})")


def _call(fn, what, device, *args):
    """fn(*args, stream) on torch's current stream, opening the engine first
    where nothing has."""
    stream = torch._C._cuda_getCurrentRawStream(device) or STREAM_DEFAULT
    rc = fn(*args, stream)
    if rc == STATE:
        Engine(device)
        rc = fn(*args, stream)
    if rc != OK:
        _raise(rc, what)


def _need(ok, what):
    if not ok:
        raise ValueError(what)


def _type(t, what):
    _need(t.is_cuda, f"{what} is on the GPU")
    code = _TYPES.get(t.dtype)
    _need(code is not None, f"{what} is float32, float16 or bfloat16")
    return code


def _row(t, what):
    """(strides, address) of a tensor whose last axis is contiguous."""
    s = t.stride()
    _need(s[-1] == 1 or t.shape[-1] == 1, f"{what}'s last axis is contiguous")
    return s


def _ints(t, n, what):
    """The address of an int32 tensor of n elements."""
    if t is None:
        return None
    _need(t.is_cuda and t.dtype == torch.int32 and t.is_contiguous() and t.numel() == n,
          f"{what} is a contiguous int32 tensor of {n} on the GPU")
    return t.data_ptr()


def _scratch(bytes_, device):
    return torch.empty(bytes_, dtype=torch.uint8, device=device) if bytes_ else None


def delta_rule(q, k, v, g, beta, state_in=None, state_out=None, *, scale=None, offsets=None, slots=None,
               max_tokens=None, normalize=False, out=None, status=None):
    """The gated delta rule, o [tokens, heads, value_dim] of
        u = beta (v - a S^T k);  S <- a S + k u^T;  o = scale S^T q,  a = exp(g)
    q, k [tokens, key_heads, key_dim], v [tokens, heads, value_dim], g and beta
    [tokens, heads] fp32. normalize: q and k are divided by sqrt(sum of squares
    + 1e-6) first; scale: key_dim ** -0.5 unless given.

    offsets (int32, sequences + 1): sequence i is tokens offsets[i] ..
    offsets[i+1]-1, at most max_tokens (default: all tokens; the work is laid
    out for it). Without offsets there are tokens / max_tokens sequences (one
    unless max_tokens is given). state_in / state_out: pools [rows, heads,
    key_dim, value_dim] fp32, the same tensor to update in place; None: from
    zeros / dropped. slots (int32, sequences): the pool row of each sequence,
    -1 to skip one; default row i."""
    code = _type(v, "v")
    _need(q.dim() == 3 and k.shape == q.shape and v.dim() == 3 and v.shape[0] == q.shape[0],
          "q and k are [tokens, key_heads, key_dim], v [tokens, heads, value_dim]")
    _need(q.dtype == v.dtype and k.dtype == v.dtype and q.is_cuda and k.is_cuda, "q, k and v have one type and device")
    tokens, key_heads, key_dim = q.shape
    _, heads, value_dim = v.shape
    _need(key_dim > 0, "key_dim is positive")
    for t, what in ((g, "g"), (beta, "beta")):
        _need(t.dtype == torch.float32 and t.is_cuda and t.shape == (tokens, heads), f"{what} is fp32 [tokens, heads]")
    if max_tokens is None:
        max_tokens = tokens
    if offsets is not None:
        sequences = offsets.numel() - 1
        _need(sequences >= 0, "offsets has sequences + 1 elements")
    else:
        _need(tokens == 0 or (max_tokens and tokens % max_tokens == 0), "without offsets, max_tokens divides tokens")
        sequences = tokens // max_tokens if tokens else 0
    rows = None
    for s, what in ((state_in, "state_in"), (state_out, "state_out")):
        if s is None:
            continue
        _need(s.dtype == torch.float32 and s.is_cuda and s.is_contiguous() and s.dim() == 4
              and s.shape[1:] == (heads, key_dim, value_dim),
              f"{what} is a contiguous fp32 [rows, heads, key_dim, value_dim]")
        _need(rows is None or rows == s.shape[0], "both state pools have the same rows")
        rows = s.shape[0]
    if rows is None:
        rows = sequences
    if out is None:
        out = torch.empty_like(v, memory_format=torch.contiguous_format)
    else:
        _need(out.shape == v.shape and out.dtype == v.dtype and out.is_cuda, "out is like v")
    qs, ks, vs, os_ = _row(q, "q"), _row(k, "k"), _row(v, "v"), _row(out, "out")
    gs, bs = _row(g, "g"), _row(beta, "beta")
    r = DeltaRequest(sequences, tokens, max_tokens, key_heads, heads, key_dim, value_dim, code,
                     DELTA_NORMALIZE if normalize else 0, rows, key_dim ** -0.5 if scale is None else scale,
                     q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), beta.data_ptr(), out.data_ptr(),
                     qs[0], qs[1], ks[0], ks[1], vs[0], vs[1], os_[0], os_[1], gs[0], bs[0],
                     _ints(offsets, sequences + 1, "offsets"), _ints(slots, sequences, "slots"),
                     None if state_in is None else state_in.data_ptr(),
                     None if state_out is None else state_out.data_ptr(), _ints(status, 1, "status"))
    L, at = lib(), C.addressof(r)
    n = L.fr_hip_delta_workspace(at)
    w = _scratch(n, v.device)
    _call(L.fr_hip_delta_rule, "fr_hip_delta_rule", v.device.index, at, w.data_ptr() if n else None, n)
    return out


def q4_product(x, codes, scales, zeros=None, *, out=None):
    """y[t, n] = sum_k x[t, k] (code[n, k] - zero[n, k // group]) scale[n, k // group].
    x [tokens, cols]; codes uint8 [rows, cols / 2], byte j holding code 2j low
    and 2j+1 high; scales fp16 or bf16 [rows, cols / group], zeros uint8 of the
    same shape or None (8). group is cols / scales' columns: 32, 64 or 128."""
    code = _type(x, "x")
    _need(x.dim() == 2 and codes.dim() == 2 and scales.dim() == 2, "x, codes and scales are matrices")
    tokens, cols = x.shape
    rows, groups = scales.shape
    _need(codes.dtype == torch.uint8 and codes.is_cuda and codes.is_contiguous() and codes.shape[0] == rows
          and codes.shape[1] * 2 == cols, "codes is a contiguous uint8 [rows, cols / 2]")
    _need(scales.dtype in (torch.float16, torch.bfloat16) and scales.is_cuda and scales.is_contiguous(),
          "scales is a contiguous fp16 or bf16 [rows, cols / group]")
    _need(groups > 0 and cols % groups == 0, "scales' columns divide cols")
    if zeros is not None:
        _need(zeros.dtype == torch.uint8 and zeros.is_cuda and zeros.is_contiguous() and zeros.shape == scales.shape,
              "zeros is a contiguous uint8 tensor like scales")
    if out is None:
        out = torch.empty((tokens, rows), dtype=x.dtype, device=x.device)
    else:
        _need(out.shape == (tokens, rows) and out.dtype == x.dtype and out.is_cuda, "out is [tokens, rows] of x's type")
    xs, ys = _row(x, "x"), _row(out, "out")
    r = Q4Request(tokens, rows, cols, cols // groups, code, _TYPES[scales.dtype], x.data_ptr(), codes.data_ptr(),
                  scales.data_ptr(), None if zeros is None else zeros.data_ptr(), out.data_ptr(), xs[0], ys[0])
    L, at = lib(), C.addressof(r)
    n = L.fr_hip_q4_workspace(at)
    w = _scratch(n, x.device)
    _call(L.fr_hip_q4_product, "fr_hip_q4_product", x.device.index, at, w.data_ptr() if n else None, n)
    return out


class KVCache(NamedTuple):
    """A paged cache in 8 bits. A token's vector of one head is dim e4m3 codes
    and one exponent byte E, each value code * 2**(E - 127). Any tuple of these
    four tensors serves."""
    k_codes: torch.Tensor   # uint8 [pages, heads, page, dim]
    v_codes: torch.Tensor   # uint8 [pages, heads, page / 16, dim, 16]: blocks of 16 tokens, tokens last
    k_exp: torch.Tensor     # uint8 [pages, heads, page]
    v_exp: torch.Tensor

    @classmethod
    def empty(cls, pages, heads, page, dim, device="cuda"):
        kw = {"dtype": torch.uint8, "device": device}
        return cls(torch.empty(pages, heads, page, dim, **kw), torch.empty(pages, heads, page // 16, dim, 16, **kw),
                   torch.empty(pages, heads, page, **kw), torch.empty(pages, heads, page, **kw))


def _cache(cache):
    k, v, ke, ve = cache
    _need(k.dim() == 4, "k_codes is [pages, heads, page, dim]")
    pages, heads, page, dim = k.shape
    _need(v.shape == (pages, heads, page // 16, dim, 16) and page % 16 == 0,
          "v_codes is [pages, heads, page / 16, dim, 16]")
    _need(ke.shape == (pages, heads, page) and ve.shape == ke.shape, "k_exp and v_exp are [pages, heads, page]")
    for t in cache:
        _need(t.dtype == torch.uint8 and t.is_cuda and t.is_contiguous(), "the cache is of contiguous uint8 tensors")
    return CacheRequest(pages, heads, page, dim, k.data_ptr(), v.data_ptr(), ke.data_ptr(), ve.data_ptr())


def _tokens(c, k, v, slots, status):
    t = v if k is None else k
    code = _type(t, "k and v")
    tokens = t.shape[0]
    at = []
    for x in (k, v):
        if x is None:
            at.append((None, (0, 0)))
            continue
        _need(x.dim() == 3 and x.shape == (tokens, c.heads, c.dim) and x.dtype == t.dtype and x.is_cuda,
              "k and v are [tokens, heads, dim] of one type")
        at.append((x.data_ptr(), _row(x, "k and v")))
    (kp, ks), (vp, vs) = at
    return TokensRequest(c, tokens, code, kp, vp, ks[0], ks[1], vs[0], vs[1], _ints(slots, tokens, "slots"),
                         _ints(status, 1, "status"))


def kv_append(cache, k, v, slots, *, status=None):
    """Writes token t's k and v [tokens, heads, dim] to place slots[t] = page
    number * page + place in it (int32, distinct; -1: skipped)."""
    r = _tokens(_cache(cache), k, v, slots, status)
    _call(lib().fr_hip_kv_append, "fr_hip_kv_append", k.device.index, C.addressof(r))


def kv_read(cache, slots, dtype=torch.bfloat16, *, status=None):
    """The values held at slots as (k, v) [tokens, heads, dim]; zeros for -1."""
    c = _cache(cache)
    shape = (slots.numel(), c.heads, c.dim)
    k = torch.empty(shape, dtype=dtype, device=slots.device)
    v = torch.empty(shape, dtype=dtype, device=slots.device)
    r = _tokens(c, k, v, slots, status)
    _call(lib().fr_hip_kv_read, "fr_hip_kv_read", k.device.index, C.addressof(r))
    return k, v


def kv_attend(cache, q, table, lengths, *, scale=None, max_context=None, out=None, status=None):
    """Attention of each sequence's last tokens over its cache. q [sequences *
    burst, heads, dim], burst 1 to 8; sequence i has lengths[i] tokens, these
    included, in pages table[i, 0 ..] (int32 [sequences, pages a row]); token b
    of its burst sees the first lengths[i] - burst + b + 1. max_context bounds
    the lengths (default: all that a table row holds). scale: dim ** -0.5
    unless given."""
    code = _type(q, "q")
    c = _cache(cache)
    _need(q.dim() == 3 and q.shape[2] == c.dim, "q is [sequences * burst, heads, dim]")
    _need(table.dim() == 2 and table.dtype == torch.int32 and table.is_cuda and (table.stride(1) == 1 or
          table.shape[1] <= 1), "table is an int32 matrix")
    sequences = table.shape[0]
    _need(q.shape[0] % sequences == 0 if sequences else q.shape[0] == 0, "q has the same burst of every sequence")
    most = table.shape[1] * c.page
    if max_context is None:
        max_context = most
    _need(0 <= max_context <= most, "max_context is within a table row's pages")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    else:
        _need(out.shape == q.shape and out.dtype == q.dtype and out.is_cuda, "out is like q")
    if not sequences or not q.shape[0]:
        return out
    qs, os_ = _row(q, "q"), _row(out, "out")
    r = QueryRequest(c, sequences, q.shape[0] // sequences, q.shape[1], max_context, code,
                     max(table.stride(0), table.shape[1]) if sequences == 1 else table.stride(0),
                     c.dim ** -0.5 if scale is None else scale, q.data_ptr(), out.data_ptr(), qs[0], qs[1], os_[0],
                     os_[1], table.data_ptr(), _ints(lengths, sequences, "lengths"), _ints(status, 1, "status"))
    L, at = lib(), C.addressof(r)
    n = L.fr_hip_kv_workspace(at)
    w = _scratch(n, q.device)
    _call(L.fr_hip_kv_attend, "fr_hip_kv_attend", q.device.index, at, w.data_ptr() if n else None, n)
    return out

