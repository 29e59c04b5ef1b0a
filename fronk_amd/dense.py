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


# A call of one token is bounded by the host, so what is checked on every call
# is checked in place, and messages are made only for a refusal.

def _type(t, what):
    code = _TYPES.get(t.dtype)
    if code is None or not t.is_cuda:
        raise ValueError(f"{what} is float32, float16 or bfloat16, on the GPU")
    return code


def _row(t, what):
    """The strides of a tensor whose last axis is contiguous."""
    s = t.stride()
    if s[-1] != 1 and t.shape[-1] != 1:
        raise ValueError(f"{what}'s last axis is contiguous")
    return s


def _ints(t, n, what):
    """The address of an int32 tensor of n elements."""
    if t is None:
        return None
    if t.dtype is not torch.int32 or t.numel() != n or not t.is_cuda or not t.is_contiguous():
        raise ValueError(f"{what} is a contiguous int32 tensor of {n} on the GPU")
    return t.data_ptr()


def _pool(s, heads, key_dim, value_dim, what):
    """(address, rows) of a state pool."""
    if s is None:
        return None, None
    shape = s.shape
    if (len(shape) != 4 or shape[1:] != (heads, key_dim, value_dim) or s.dtype is not torch.float32
            or not s.is_cuda or not s.is_contiguous()):
        raise ValueError(f"{what} is a contiguous fp32 [rows, heads, key_dim, value_dim]")
    return s.data_ptr(), shape[0]


def _run(name, workspace, request, device):
    """The call with the workspace that it asks for."""
    L, at = lib(), C.addressof(request)
    n = getattr(L, workspace)(at)
    if n:
        w = torch.empty(n, dtype=torch.uint8, device=device)
        _call(getattr(L, name), name, device.index, at, w.data_ptr(), n)
    else:
        _call(getattr(L, name), name, device.index, at, None, 0)


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
    qshape, vshape = q.shape, v.shape
    if len(qshape) != 3 or k.shape != qshape or len(vshape) != 3 or vshape[0] != qshape[0]:
        raise ValueError("q and k are [tokens, key_heads, key_dim], v [tokens, heads, value_dim]")
    if q.dtype is not v.dtype or k.dtype is not v.dtype or not q.is_cuda or not k.is_cuda:
        raise ValueError("q, k and v have one type and device")
    tokens, key_heads, key_dim = qshape
    _, heads, value_dim = vshape
    if key_dim <= 0:
        raise ValueError("key_dim is positive")
    scalars = (tokens, heads)
    if (g.shape != scalars or beta.shape != scalars or g.dtype is not torch.float32
            or beta.dtype is not torch.float32 or not g.is_cuda or not beta.is_cuda):
        raise ValueError("g and beta are fp32 [tokens, heads]")
    if max_tokens is None:
        max_tokens = tokens
    if offsets is not None:
        sequences = offsets.numel() - 1
        if sequences < 0:
            raise ValueError("offsets has sequences + 1 elements")
    else:
        _need(tokens == 0 or (max_tokens and tokens % max_tokens == 0), "without offsets, max_tokens divides tokens")
        sequences = tokens // max_tokens if tokens else 0
    before, rows = _pool(state_in, heads, key_dim, value_dim, "state_in")
    if state_out is state_in:
        after = before
    else:
        after, others = _pool(state_out, heads, key_dim, value_dim, "state_out")
        if rows is None:
            rows = others
        elif others is not None and others != rows:
            raise ValueError("both state pools have the same rows")
    if rows is None:
        rows = sequences
    device = v.device
    if out is None:
        out = torch.empty(vshape, dtype=v.dtype, device=device)
    elif out.shape != vshape or out.dtype is not v.dtype or not out.is_cuda:
        raise ValueError("out is like v")
    qs, ks, vs, os_ = _row(q, "q"), _row(k, "k"), _row(v, "v"), _row(out, "out")
    gs, bs = _row(g, "g"), _row(beta, "beta")
    r = DeltaRequest(sequences, tokens, max_tokens, key_heads, heads, key_dim, value_dim, code,
                     DELTA_NORMALIZE if normalize else 0, rows, key_dim ** -0.5 if scale is None else scale,
                     q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), beta.data_ptr(), out.data_ptr(),
                     qs[0], qs[1], ks[0], ks[1], vs[0], vs[1], os_[0], os_[1], gs[0], bs[0],
                     _ints(offsets, sequences + 1, "offsets"), _ints(slots, sequences, "slots"), before, after,
                     _ints(status, 1, "status"))
    _run("fr_hip_delta_rule", "fr_hip_delta_workspace", r, device)
    return out


def q4_product(x, codes, scales, zeros=None, *, out=None):
    """y[t, n] = sum_k x[t, k] (code[n, k] - zero[n, k // group]) scale[n, k // group].
    x [tokens, cols]; codes uint8 [rows, cols / 2], byte j holding code 2j low
    and 2j+1 high; scales fp16 or bf16 [rows, cols / group], zeros uint8 of the
    same shape or None (8). group is cols / scales' columns: 32, 64 or 128."""
    code = _type(x, "x")
    xshape, wshape, sshape = x.shape, codes.shape, scales.shape
    if len(xshape) != 2 or len(wshape) != 2 or len(sshape) != 2:
        raise ValueError("x, codes and scales are matrices")
    tokens, cols = xshape
    rows, groups = sshape
    if (wshape[0] != rows or wshape[1] * 2 != cols or codes.dtype is not torch.uint8 or not codes.is_cuda
            or not codes.is_contiguous()):
        raise ValueError("codes is a contiguous uint8 [rows, cols / 2]")
    scale_type = scales.dtype
    if scale_type not in (torch.float16, torch.bfloat16) or not scales.is_cuda or not scales.is_contiguous():
        raise ValueError("scales is a contiguous fp16 or bf16 [rows, cols / group]")
    if groups <= 0 or cols % groups:
        raise ValueError("scales' columns divide cols")
    if zeros is not None and (zeros.dtype is not torch.uint8 or zeros.shape != sshape or not zeros.is_cuda
                              or not zeros.is_contiguous()):
        raise ValueError("zeros is a contiguous uint8 tensor like scales")
    device = x.device
    if out is None:
        out = torch.empty((tokens, rows), dtype=x.dtype, device=device)
    elif out.shape != (tokens, rows) or out.dtype is not x.dtype or not out.is_cuda:
        raise ValueError("out is [tokens, rows] of x's type")
    r = Q4Request(tokens, rows, cols, cols // groups, code, _TYPES[scale_type], x.data_ptr(), codes.data_ptr(),
                  scales.data_ptr(), None if zeros is None else zeros.data_ptr(), out.data_ptr(), _row(x, "x")[0],
                  _row(out, "out")[0])
    _run("fr_hip_q4_product", "fr_hip_q4_workspace", r, device)
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
    shape = k.shape
    if len(shape) != 4:
        raise ValueError("k_codes is [pages, heads, page, dim]")
    pages, heads, page, dim = shape
    if page % 16 or v.shape != (pages, heads, page // 16, dim, 16):
        raise ValueError("v_codes is [pages, heads, page / 16, dim, 16]")
    if ke.shape != shape[:3] or ve.shape != shape[:3]:
        raise ValueError("k_exp and v_exp are [pages, heads, page]")
    for t in (k, v, ke, ve):
        if t.dtype is not torch.uint8 or not t.is_cuda or not t.is_contiguous():
            raise ValueError("the cache is of contiguous uint8 tensors")
    return CacheRequest(pages, heads, page, dim, k.data_ptr(), v.data_ptr(), ke.data_ptr(), ve.data_ptr())


def _tokens(c, k, v, slots, status):
    """The request for k and v, two tensors [tokens, heads, dim] alike."""
    code = _type(k, "k and v")
    shape = k.shape
    if (len(shape) != 3 or shape[1] != c.heads or shape[2] != c.dim or v.shape != shape or v.dtype is not k.dtype
            or not v.is_cuda):
        raise ValueError("k and v are [tokens, heads, dim] of one type")
    ks, vs = _row(k, "k and v"), _row(v, "k and v")
    return TokensRequest(c, shape[0], code, k.data_ptr(), v.data_ptr(), ks[0], ks[1], vs[0], vs[1],
                         _ints(slots, shape[0], "slots"), _ints(status, 1, "status"))


def kv_append(cache, k, v, slots, *, status=None):
    """Writes token t's k and v [tokens, heads, dim] to place slots[t] = page
    number * page + place in it (int32, distinct; -1: skipped)."""
    r = _tokens(_cache(cache), k, v, slots, status)
    _call(lib().fr_hip_kv_append, "fr_hip_kv_append", k.device.index, C.addressof(r))


def kv_read(cache, slots, dtype=torch.bfloat16, *, status=None):
    """The values held at slots as (k, v) [tokens, heads, dim]; zeros for -1."""
    c = _cache(cache)
    k, v = torch.empty((2, slots.numel(), c.heads, c.dim), dtype=dtype, device=slots.device)
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
    if q.dim() != 3 or q.shape[2] != c.dim:
        raise ValueError("q is [sequences * burst, heads, dim]")
    if (table.dim() != 2 or table.dtype is not torch.int32 or not table.is_cuda
            or (table.stride(1) != 1 and table.shape[1] > 1)):
        raise ValueError("table is an int32 matrix")
    sequences = table.shape[0]
    _need(q.shape[0] % sequences == 0 if sequences else q.shape[0] == 0, "q has the same burst of every sequence")
    most = table.shape[1] * c.page
    if max_context is None:
        max_context = most
    _need(0 <= max_context <= most, "max_context is within a table row's pages")
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    elif out.shape != q.shape or out.dtype is not q.dtype or not out.is_cuda:
        raise ValueError("out is like q")
    if not sequences or not q.shape[0]:
        return out
    qs, os_ = _row(q, "q"), _row(out, "out")
    r = QueryRequest(c, sequences, q.shape[0] // sequences, q.shape[1], max_context, code,
                     max(table.stride(0), table.shape[1]) if sequences == 1 else table.stride(0),
                     c.dim ** -0.5 if scale is None else scale, q.data_ptr(), out.data_ptr(), qs[0], qs[1], os_[0],
                     os_[1], table.data_ptr(), _ints(lengths, sequences, "lengths"), _ints(status, 1, "status"))
    _run("fr_hip_kv_attend", "fr_hip_kv_workspace", r, q.device)
    return out
