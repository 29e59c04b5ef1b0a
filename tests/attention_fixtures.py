"""Attention of prompts and of trees in 64 bits on the CPU, and what outputs may be
off (not collected by pytest)."""
import torch

from dense_fixtures import HALF, U


def softmax_rows(q, k, v, seen, scale):
    """(o, sum of weights times |v|, largest sum of a score's |terms|) of rows
    q [rows][heads][dim] over k, v [keys][key heads][dim], where seen [rows][keys];
    zeros where nothing is. In 64 bits."""
    q, k, v = q.double(), k.double(), v.double()
    r = q.shape[1] // k.shape[1]
    k, v = k.repeat_interleave(r, 1), v.repeat_interleave(r, 1)
    if k.shape[0] == 0:
        return torch.zeros_like(q), torch.zeros_like(q), torch.zeros(q.shape[0], q.shape[1], 1, dtype=torch.float64)
    hide = ~seen[None]
    s = (scale * (q.transpose(0, 1) @ k.permute(1, 2, 0).contiguous())).masked_fill(hide, -torch.inf)
    p = torch.nan_to_num(torch.softmax(s, -1), nan=0.0) if not torch.isnan(s).any() else torch.softmax(s, -1)
    terms = abs(scale) * (q.abs().transpose(0, 1) @ k.abs().permute(1, 2, 0).contiguous()).masked_fill(hide, 0)
    o, size = (p @ x.transpose(0, 1).contiguous() for x in (v, v.abs()))
    return o.transpose(0, 1), size.transpose(0, 1), terms.amax(-1).T[..., None]


def prompt(q, k, v, lens, k_lens, scale):
    """Packed prompts, as softmax_rows."""
    parts, t, s = [], 0, 0
    for n, m in zip(lens, k_lens):
        seen = torch.arange(m) <= m - n + torch.arange(n)[:, None]
        parts.append(softmax_rows(q[t:t + n], k[s:s + m], v[s:s + m], seen, scale))
        t, s = t + n, s + m
    return tuple(torch.cat(x) for x in zip(*parts))


def attend_tolerance(o, size, terms, dtype, weights, dim, keys, largest):
    """What outputs may be off: their own rounding; a weight's, `weights` relative to it
    (in fp16 at least 2^-25 of the row's largest, times the largest value of each key);
    and fp32's: a score's sum over dim terms and two factors, its exp2 (2^-22), and sums
    over the keys. What a weight is off by, outputs are off by twice, as the sum
    of weights is off too."""
    delta = U * ((dim + 2) * terms + keys) + 2.0 ** -22
    subnormal = 2.0 ** -25 * keys * largest if dtype == torch.float16 else 0.0
    return HALF[dtype] * o.abs() + (weights + 2 * delta) * size + subnormal


def tree(q, k, v, masks, lens, scale):
    """Trees, as softmax_rows: k and v lists of [tokens][heads][dim] per sequence, its drafts
    the last of them."""
    parts, t = [], 0
    for n, x, y in zip(lens, k, v):
        m = x.shape[0]
        seen = torch.ones(n, m, dtype=torch.bool)
        for b in range(n):
            for j in range(n):
                seen[b, m - n + j] = bool((masks[t + b] >> j) & 1)
        parts.append(softmax_rows(q[t:t + n], x, y, seen, scale))
        t += n
    return tuple(torch.cat(x) for x in zip(*parts))


def random_tree(rand, drafts):
    """Words of `drafts` drafts, each behind one of those before it or a beginning."""
    seen = []
    for b in range(drafts):
        parent = rand.randint(max(-1, b - 4), b - 1)
        seen.append((seen[parent] if parent >= 0 else 0) | 1 << b)
    return seen


def words(masks):
    return torch.tensor([x - (1 << 64) if x >> 63 else x for x in masks], dtype=torch.int64)
