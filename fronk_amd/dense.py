"""The dense operators over torch tensors: thin calls of the C ABI
(include/fronk_hip.h, through host/dense_module.cpp), enqueued on torch's current
stream, no compute and no fallback of their own. Tensors are on the open engine's
device (fr_hip_open; the first call here opens theirs, and tensors on another one
are refused) and may have any strides but for a contiguous last axis.

  delta_rule   the gated delta rule, decode bursts to prompts
  q4_product   products with 4-bit weights and group scales
  KVCache, kv_append, kv_read, kv_attend   the paged 8-bit key/value cache

They have no backward pass: a tensor that requires a gradient is refused unless
under torch.no_grad() (or inference_mode), one with a forward-mode tangent always.

A refused call raises ValueError before anything is enqueued. What only the
device can see (offsets, slots, pages, lengths) is bounds-checked there: a bad
entry reads nothing, leaves what it would write as it was (zeros in kv_read's and
kv_attend's outputs) and sets its bit (BAD_*) in `status`, an int32 tensor of one
element that the caller clears. Call once before capturing a graph.
"""
import ctypes as C
from typing import NamedTuple

import torch

from . import Engine

F32, F16, BF16 = 0, 1, 2
BAD_OFFSET, BAD_SLOT, BAD_PAGE, BAD_LENGTH = 1, 2, 4, 8
DELTA_NORMALIZE = 1

# The C ABI's request structures.
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


class _Missing:
    def __getattr__(self, name):
        raise RuntimeError("fronk_amd/_dense.so is missing: run __graft_entry__.build()")


try:
    from . import _dense
    _dense.bind(Engine, torch._C._cuda_getCurrentRawStream)
except ImportError:
    _dense = _Missing()


def delta_rule(q, k, v, g, beta, state_in=None, state_out=None, *, scale=None, offsets=None, slots=None,
               max_tokens=None, normalize=False, out=None, status=None):
    """The gated delta rule, o [tokens, heads, value_dim] of
        u = beta (v - a S^T k);  S <- a S + k u^T;  o = scale S^T q,  a = exp(g)
    q, k [tokens, key_heads, key_dim], v [tokens, heads, value_dim], g and beta
    [tokens, heads] fp32. normalize: q and k are divided by sqrt(sum of squares
    + 1e-6) first; scale: key_dim ** -0.5 unless given. Non-finite inputs reach
    no token before theirs.

    offsets (int32, sequences + 1): sequence i is tokens offsets[i] ..
    offsets[i+1]-1, at most max_tokens (default: all tokens; the work is laid
    out for it). Without offsets there are tokens / max_tokens sequences (one
    unless max_tokens is given). state_in / state_out: pools [rows, heads,
    key_dim, value_dim] fp32, the same tensor to update in place; None: from
    zeros / dropped. slots (int32, sequences): the pool row of each sequence,
    -1 to skip one; default row i. out shares no memory with an input."""
    return _dense.delta_rule(q, k, v, g, beta, state_in, state_out, scale, offsets, slots, max_tokens, normalize, out,
                             status)


def q4_product(x, codes, scales, zeros=None, *, out=None):
    """y[t, n] = sum_k x[t, k] (code[n, k] - zero[n, k // group]) scale[n, k // group].
    x [tokens, cols]; codes uint8 [rows, cols / 2], byte j holding code 2j low
    and 2j+1 high; scales fp16 or bf16 [rows, cols / group], zeros uint8 of the
    same shape or None (8). group is cols / scales' columns: 32, 64 or 128."""
    return _dense.q4_product(x, codes, scales, zeros, out)


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


def kv_append(cache, k, v, slots, *, status=None):
    """Writes token t's k and v [tokens, heads, dim] to place slots[t] = page
    number * page + place in it (int32, distinct; -1: skipped)."""
    _dense.kv_append(cache, k, v, slots, status)


def kv_read(cache, slots, dtype=torch.bfloat16, *, status=None):
    """The values held at slots as (k, v) [tokens, heads, dim]; zeros for -1."""
    return _dense.kv_read(cache, slots, dtype, status)


def kv_attend(cache, q, table, lengths, *, scale=None, max_context=None, out=None, status=None):
    """Attention of each sequence's last tokens over its cache. q [sequences *
    burst, heads, dim], burst 1 to 8; sequence i has lengths[i] tokens, these
    included, in pages table[i, 0 ..] (int32 [sequences, pages a row]); token b
    of its burst sees the first lengths[i] - burst + b + 1. max_context bounds
    the lengths (default: all that a table row holds). scale: dim ** -0.5
    unless given."""
    return _dense.kv_attend(cache, q, table, lengths, scale, max_context, out, status)
