"""The operators of an attention layer around its 8-bit paged cache that are
timed, through their public entry points.

What a server does in such a layer beside appending tokens to the cache and
attending to it with bursts (perf/operators.py):

  rotary  fronk_amd.dense.rotary: positions turned into q and k, both layouts of
          pairs, all of a head or its first part, scaled for long contexts;
  prompt  fronk_amd.dense.prompt_attend: causal attention of packed prompts of
          unequal lengths over their own keys, or over earlier ones too;
  tree    fronk_amd.dense.kv_attend_tree: a tree of drafted tokens over the
          cache, each seeing what came before the drafts and its own ancestors;
  move    fronk_amd.dense.kv_move: accepted drafts moved together in the cache;
  copy    fronk_amd.dense.kv_copy: pages of the cache forked.

`run` in its plain form computes the same in 32 bits from elementary torch
operations (positions' angles in 64). The layout of the cache is the public one
that fronk_amd.dense documents, so both forms take the same state.
"""
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
MOST_MOVES = 64


def _rotary(name, tokens, heads, kv_heads, dim, rotated, interleaved, scaled, dtype):
    return {"name": name, "op": "rotary", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "rotated": rotated, "interleaved": interleaved, "scaled": scaled, "dtype": dtype}


def _prompt(name, seqs, tokens, earlier, heads, kv_heads, dim, dtype, ragged=False):
    return {"name": name, "op": "prompt", "seqs": seqs, "tokens": tokens, "earlier": earlier, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "ragged": ragged}


def _tree(name, seqs, drafts, context, heads, kv_heads, dim, page, dtype, ragged=False):
    return {"name": name, "op": "tree", "seqs": seqs, "drafts": drafts, "context": context, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype, "ragged": ragged}


def _move(name, groups, moves, kv_heads, dim, page):
    return {"name": name, "op": "move", "groups": groups, "moves": moves, "kv_heads": kv_heads, "dim": dim,
            "page": page}


def _copy(name, pages, kv_heads, dim, page):
    return {"name": name, "op": "copy", "pages": pages, "kv_heads": kv_heads, "dim": dim, "page": page}


def listed():
    return [
        # One user's next token; a quarter of each head has positions.
        _rotary("rotary_token", 1, 16, 2, 256, 64, False, False, "bf16"),
        # The longest prefill chunk, far into a context that was scaled.
        _rotary("rotary_chunk", 4096, 20, 4, 128, 128, True, True, "f16"),
        # The longest prefill chunk of one prompt.
        _prompt("prompt_long", 1, 4096, 0, 16, 2, 256, "bf16"),
        # Prompts of unequal lengths packed into one call, odd groups of heads.
        _prompt("prompt_packed", 7, 1531, 0, 20, 4, 128, "f16", ragged=True),
        # A later chunk of a long prompt over all that came before.
        _prompt("prompt_chunk", 1, 512, 7680, 32, 4, 128, "bf16"),
        # Many short questions, 32-bit activations.
        _prompt("prompt_short", 33, 61, 0, 6, 2, 64, "f32", ragged=True),
        # One stream with a small tree over a long context.
        _tree("tree_one", 1, 15, 32768, 16, 2, 256, 64, "bf16"),
        # A serving batch with trees of unequal sizes over unequal contexts.
        _tree("tree_batch", 24, 61, 8192, 16, 4, 128, 32, "f16", ragged=True),
        # One stream's accepted path.
        _move("move_path", 1, 6, 2, 256, 64),
        # A serving batch's accepted paths.
        _move("move_batch", 128, 24, 8, 128, 16),
        # A stream forked: its last pages.
        _copy("copy_fork", 3, 2, 256, 64),
        # Many streams forked at once, or a cache put in order.
        _copy("copy_pages", 1024, 2, 256, 64),
    ]


def _log_int(rng, lo, hi):
    hi = max(lo, int(hi))
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rotary", "rotary", "prompt", "prompt", "prompt", "tree", "tree", "move", "copy"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    kv_heads = rng.choice([1, 2, 2, 3, 4, 8])
    dim = rng.choice([64, 128, 128, 256])
    page = rng.choice([16, 32, 64, 128])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 7, 8])
    if op == "rotary":
        rotated = dim if rng.random() < 0.5 else 2 * rng.randint(1, dim // 2)
        tokens = _log_int(rng, 1, min(8192, 4096 * 24 * 128 // ((heads + kv_heads) * dim)))
        c = _rotary("", tokens, heads, kv_heads, dim, rotated, rng.random() < 0.5, rng.random() < 0.5, dtype)
    elif op == "prompt":
        # (32 bits: a quarter of the work, as the plain form's scores and sums of
        # all types are 32 bits wide and the listed largest one is of 16)
        most = 16 * 256 * 4096 * 2048 // (4 if dtype == "f32" else 1) // (heads * dim)
        seqs = _log_int(rng, 1, 48)
        tokens = _log_int(rng, 1, min(4096, math.isqrt(2 * most // seqs)))
        earlier = 0 if rng.random() < 0.6 else _log_int(rng, 1, min(16384, max(1, most // (seqs * tokens) - tokens)))
        c = _prompt("", seqs, tokens, earlier, heads, kv_heads, dim, dtype, rng.random() < 0.6)
    elif op == "tree":
        seqs = _log_int(rng, 1, 32)
        drafts = _log_int(rng, 1, 64)
        heads = min(heads, kv_heads * 4) if drafts > 32 else heads
        most = 24 * 61 * 8192 * 16 * 128 // (seqs * drafts * heads * dim)
        most = min(most, 24 * 8192 * 4 * 128 // (seqs * kv_heads * dim), 65536)
        c = _tree("", seqs, drafts, drafts + _log_int(rng, 1, max(1, most - drafts)), heads, kv_heads, dim, page,
                  dtype, rng.random() < 0.6)
    elif op == "move":
        c = _move("", _log_int(rng, 1, 128), rng.randint(1, MOST_MOVES), kv_heads, dim, page)
    else:
        c = _copy("", _log_int(rng, 1, 1024 * 2 * 256 * 64 // (kv_heads * dim * page)), kv_heads, dim, page)
    del c["name"]
    return c


# ------------------------------------------------------------------ inputs

def _spread(low, top, n, ragged):
    """n whole numbers from the case alone: all `top`, or spread evenly between."""
    if not ragged or n == 1:
        return [top] * n
    return [low + ((7 * i + 3) % n) * (top - low) // (n - 1) for i in range(n)]


def _starts(lens):
    return [sum(lens[:i]) for i in range(len(lens) + 1)]


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _frequencies(rotated, scaled):
    """In radians a position, 64 bits. Scaled: the context is 32 times as long as
    the 4096 positions that the frequencies were learnt for; what turns less than
    once in those is slowed by 32, what turns more than 32 times is kept, and in
    between goes a ramp over the number of turns. q and k grow by 1 + ln(32) / 10."""
    f = 10000.0 ** (-torch.arange(0, rotated, 2, dtype=torch.float64, device="cuda") / rotated)
    if not scaled:
        return f, 1.0
    kept = ((4096 * f / (2 * math.pi) - 1) / 31).clamp(0, 1)
    return f * (kept + (1 - kept) / 32), 1 + 0.1 * math.log(32)


def _prepare_rotary(case, rand):
    t, h, hk, d = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
    row = rand(t, (h + 2 * hk) * d).to(TYPES[case["dtype"]])    # q, k and v as one projection leaves them
    first = int(torch.randint(0, 131072 if case["scaled"] else 4096, (1,), generator=rand.host))
    f, magnitude = _frequencies(case["rotated"], case["scaled"])
    return {"q": row[:, :h * d].unflatten(1, (h, d)), "k": row[:, h * d:(h + hk) * d].unflatten(1, (hk, d)),
            "positions": torch.arange(first, first + t, dtype=torch.int32, device="cuda"), "frequencies": f,
            "magnitude": magnitude, "interleaved": case["interleaved"]}


def _prompt_lengths(case):
    n = _spread(1, case["tokens"], case["seqs"], case["ragged"])
    before = _spread(0, case["earlier"], case["seqs"], case["ragged"])
    return n, [a + b for a, b in zip(n, before)]


def _prepare_prompt(case, rand):
    n, m = _prompt_lengths(case)
    h, hk, d, dt = case["heads"], case["kv_heads"], case["dim"], TYPES[case["dtype"]]
    if case["earlier"]:
        q, k, v = rand(sum(n), h, d).to(dt), rand(sum(m), hk, d).to(dt), rand(sum(m), hk, d).to(dt)
    else:   # views of one projection's rows
        row = rand(sum(n), (h + 2 * hk) * d).to(dt)
        q, k, v = (row[:, a * d:b * d].unflatten(1, (b - a, d)) for a, b in ((0, h), (h, h + hk), (h + hk, h + 2 * hk)))
    return {"q": q, "k": k, "v": v, "offsets": _ints(_starts(n)), "k_offsets": _ints(_starts(m)),
            "max_tokens": max(n), "max_context": max(m), "scale": 2.0 * d ** -0.5}


def _empty_cache(pages, heads, page, dim):
    """The cache's four arrays (fronk_amd.dense.KVCache): K codes by token, V
    codes by blocks of 16 tokens, and the two exponents."""
    kw = {"dtype": torch.uint8, "device": "cuda"}
    return (torch.empty(pages, heads, page, dim, **kw), torch.empty(pages, heads, page // 16, dim, 16, **kw),
            torch.empty(pages, heads, page, **kw), torch.empty(pages, heads, page, **kw))


def _filled_cache(pages, heads, page, dim, rand):
    """Codes of normal values at a scale that puts their largest near 448, and
    exponents that bring them back to about one."""
    cache = _empty_cache(pages, heads, page, dim)
    for codes in cache[:2]:
        flat = codes.view(-1)
        for i in range(0, flat.numel(), 1 << 26):
            part = flat[i:i + (1 << 26)]
            part.copy_((100 * rand(part.numel())).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8))
    for e in cache[2:]:
        e.copy_(torch.randint(119, 122, e.shape, device="cuda", generator=rand.generator))
    return cache


def _tree_lengths(case):
    """Drafts, and tokens with them, of each sequence."""
    n = _spread(1, case["drafts"], case["seqs"], case["ragged"])
    before = _spread(1, case["context"] - case["drafts"], case["seqs"], case["ragged"])[::-1]
    return n, [a + b for a, b in zip(n, before)]


def _prepare_tree(case, rand):
    n, m = _tree_lengths(case)
    p, d, seqs = case["page"], case["dim"], case["seqs"]
    per = (max(m) + p - 1) // p
    chance, masks = random.Random(int(torch.randint(0, 1 << 30, (1,), generator=rand.host))), []
    for drafts in n:   # each draft follows one of the few before it, or begins a branch of its own
        seen = []
        for b in range(drafts):
            parent = chance.randint(max(-1, b - 5), b - 1)
            seen.append((seen[parent] if parent >= 0 else 0) | 1 << b)
        masks += [x - (1 << 64) if x >> 63 else x for x in seen]
    order = torch.randperm(seqs * per, device="cuda", generator=rand.generator).to(torch.int32)
    return {"q": rand(sum(n), case["heads"], d).to(TYPES[case["dtype"]]),
            "cache": _filled_cache(seqs * per, case["kv_heads"], p, d, rand),
            "tree": torch.tensor(masks, dtype=torch.int64, device="cuda"), "table": order.view(seqs, per),
            "lengths": _ints(m), "offsets": _ints(_starts(n)), "max_tokens": max(n), "max_context": max(m),
            "scale": 2.0 * d ** -0.5}


def _prepare_move(case, rand):
    g, n, p = case["groups"], case["moves"], case["page"]
    drafts = 2 * n                                   # of which n at most were accepted
    per = (drafts + p - 1) // p + 1
    order = torch.randperm(g * per, device="cuda", generator=rand.generator).view(g, per)
    first = torch.randint(0, p, (g, 1), device="cuda", generator=rand.generator)
    path = torch.rand(g, drafts, device="cuda", generator=rand.generator).argsort(1)[:, :n].sort(1).values
    kept = torch.arange(n, device="cuda").expand(g, n)
    count = torch.tensor(_spread(1, n, g, True), device="cuda")[:, None]

    def slot(place):
        at = first + place
        return torch.where(kept < count, order.gather(1, at // p) * p + at % p, -1).to(torch.int32)

    return {"cache": _filled_cache(g * per, case["kv_heads"], p, case["dim"], rand), "source": slot(path),
            "target": slot(kept)}


def _prepare_copy(case, rand):
    n = case["pages"]
    order = torch.randperm(2 * n, device="cuda", generator=rand.generator).to(torch.int32)
    return {"cache": _filled_cache(2 * n, case["kv_heads"], case["page"], case["dim"], rand),
            "source": order[:n].clone(), "target": order[n:].clone()}


class _Rand:
    """Normal values on the GPU from one seeded generator."""

    def __init__(self, seed):
        self.generator = torch.Generator(device="cuda")
        self.generator.manual_seed(seed)
        self.host = torch.Generator().manual_seed(seed)

    def __call__(self, *shape):
        return torch.randn(*shape, device="cuda", generator=self.generator)


def prepare(case, seed):
    make = {"rotary": _prepare_rotary, "prompt": _prepare_prompt, "tree": _prepare_tree, "move": _prepare_move,
            "copy": _prepare_copy}
    return {"op": case["op"], **make[case["op"]](case, _Rand(seed))}


# ------------------------------------------------------------------ one pass

def _held(cache):
    """The cache as what it stands for: e4m3 values and their powers of two."""
    return tuple(x.view(torch.float8_e4m3fn) for x in cache[:2]) + tuple(cache[2:])


def run(state):
    s = dict(state)
    op = s.pop("op")
    if own:
        from fronk_amd import dense
        if op == "rotary":
            return dense.rotary(s["q"], s["k"], s["positions"], s["frequencies"], interleaved=s["interleaved"],
                                magnitude=s["magnitude"])
        if op == "prompt":
            return dense.prompt_attend(s["q"], s["k"], s["v"], offsets=s["offsets"], k_offsets=s["k_offsets"],
                                       max_tokens=s["max_tokens"], max_context=s["max_context"], scale=s["scale"])
        if op == "tree":
            return dense.kv_attend_tree(s["cache"], s["q"], s["tree"], s["table"], s["lengths"], offsets=s["offsets"],
                                        max_tokens=s["max_tokens"], max_context=s["max_context"], scale=s["scale"])
        if op == "move":
            dense.kv_move(s["cache"], s["source"], s["target"])
        else:
            dense.kv_copy(s["cache"], s["source"], s["target"])
        return _held(s["cache"])
    return {"rotary": _plain_rotary, "prompt": _plain_prompt, "tree": _plain_tree, "move": _plain_move,
            "copy": _plain_copy}[op](**s)


def _plain_rotary(q, k, positions, frequencies, magnitude, interleaved):
    angle = positions.double()[:, None] * frequencies
    c, s = ((magnitude * x).float()[:, None] for x in (torch.cos(angle), torch.sin(angle)))
    n = frequencies.shape[0]

    def turn(x):
        y = x.float()
        a, b = (y[..., 0:2 * n:2], y[..., 1:2 * n:2]) if interleaved else (y[..., :n], y[..., n:2 * n])
        a, b = a * c - b * s, a * s + b * c
        pairs = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
        return torch.cat([pairs, y[..., 2 * n:]], -1).to(x.dtype)

    return turn(q), turn(k)


def _padded(x, offsets, most):
    """[sequence][row][...] of a packed tensor in 32 bits, zeros behind the last."""
    at = offsets[:-1, None].long() + torch.arange(most, device=x.device)
    live = at < offsets[1:, None]
    return x[torch.where(live, at, 0)].float() * live.view(live.shape + (1,) * (x.dim() - 1)), live


def _softmax_sum(q, k, v, seen, scale):
    """softmax(scale q k^T over what is seen) v; zeros where nothing is."""
    p = torch.where(seen, (q @ k.transpose(-1, -2).contiguous()) * scale, -math.inf)
    top = p.amax(-1, keepdim=True)
    p = torch.exp(p - torch.where(top > -math.inf, top, 0.0))
    total = p.sum(-1, keepdim=True)
    return (p @ v) / torch.where(total > 0, total, 1.0)


def _grouped(q, heads):
    """[sequence][token][head][dim] as [sequence][key head][its heads by tokens][dim]"""
    seqs, n, h, d = q.shape
    return q.view(seqs, n, heads, h // heads, d).permute(0, 2, 3, 1, 4).reshape(seqs, heads, h // heads * n, d)


def _ungrouped(o, n):
    seqs, heads, rows, d = o.shape
    return o.view(seqs, heads, rows // n, n, d).permute(0, 3, 1, 2, 4).reshape(seqs, n, rows // n * heads, d)


def _plain_prompt(q, k, v, offsets, k_offsets, max_tokens, max_context, scale):
    hk, per = k.shape[1], q.shape[1] // k.shape[1]
    qs, live = _padded(q, offsets, max_tokens)
    ks, vs = (_padded(x, k_offsets, max_context)[0].transpose(1, 2).contiguous() for x in (k, v))
    last = (k_offsets[1:] - k_offsets[:-1] - offsets[1:] + offsets[:-1])[:, None] + torch.arange(max_tokens, device=q.device)
    seen = torch.arange(max_context, device=q.device) <= last[..., None]
    o = _softmax_sum(_grouped(qs, hk), ks, vs, seen.repeat(1, per, 1)[:, None], scale)
    return _ungrouped(o, max_tokens)[live].to(q.dtype)


def _values(codes, exponents):
    return torch.ldexp(codes.view(torch.float8_e4m3fn).float(), exponents.int()[..., None] - 127)


def _plain_tree(q, cache, tree, table, lengths, offsets, max_tokens, max_context, scale):
    kc, vc, ke, ve = cache
    h, t = kc.shape[1], table.long()
    k = _values(kc[t], ke[t]).transpose(1, 2).flatten(2, 3)[:, :, :max_context]     # [sequence][head][token][d]
    v = _values(vc[t].transpose(-1, -2).flatten(3, 4), ve[t]).transpose(1, 2).flatten(2, 3)[:, :, :max_context]
    qs, live = _padded(q, offsets, max_tokens)
    at = torch.where(live, offsets[:-1, None].long() + torch.arange(max_tokens, device=q.device), 0)
    place = torch.arange(max_context, device=q.device) - (lengths - offsets[1:] + offsets[:-1])[:, None]   # among the drafts
    bit = (tree[at][..., None] >> place.clamp(0, 63)[:, None]) & 1
    seen = (place < 0)[:, None] | ((bit == 1) & (place < (offsets[1:] - offsets[:-1])[:, None])[:, None])
    o = _softmax_sum(_grouped(qs, h), k, v, seen.repeat(1, q.shape[1] // h, 1)[:, None], scale)
    return _ungrouped(o, max_tokens)[live].to(q.dtype)


def _plain_move(cache, source, target):
    kc, vc, ke, ve = cache
    page = kc.shape[2]
    live = source.flatten() >= 0
    (sp, sa), (tp, ta) = ((x // page, x % page) for x in (s.flatten()[live].long() for s in (source, target)))
    k, v, x, y = kc[sp, :, sa], vc[sp, :, sa // 16, :, sa % 16], ke[sp, :, sa], ve[sp, :, sa]
    kc[tp, :, ta], vc[tp, :, ta // 16, :, ta % 16], ke[tp, :, ta], ve[tp, :, ta] = k, v, x, y
    return _held(cache)


def _plain_copy(cache, source, target):
    kc, vc, ke, ve = cache
    s, t = source.long(), target.long()
    kc[t], vc[t], ke[t], ve[t] = kc[s], vc[s], ke[s], ve[s]
    return _held(cache)


def work(case):
    if case["op"] in ("move", "copy"):
        tokens = case["pages"] * case["page"] if case["op"] == "copy" else \
            sum(_spread(1, case["moves"], case["groups"], True))
        return {"bytes": 2 * tokens * case["kv_heads"] * (2 * case["dim"] + 2) + 8, "flops": 0}
    size, d, h, hk = SIZE[case["dtype"]], case["dim"], case["heads"], case["kv_heads"]
    if case["op"] == "rotary":
        rows = case["tokens"] * (h + hk)
        return {"bytes": 2 * size * rows * d + 4 * case["tokens"], "flops": 3 * rows * case["rotated"]}
    if case["op"] == "prompt":
        n, m = _prompt_lengths(case)
        pairs = sum(a * b - a * (a - 1) // 2 for a, b in zip(n, m))
        return {"bytes": size * d * 2 * (sum(n) * h + sum(m) * hk), "flops": 4 * pairs * h * d}
    n, m = _tree_lengths(case)
    pairs = sum(a * (b - a + 1) for a, b in zip(n, m))
    return {"bytes": sum(m) * hk * (2 * d + 2) + 2 * size * sum(n) * h * d, "flops": 4 * pairs * h * d}


# ------------------------------------------------------- the result in 64 bits

def _exact_rotary(s):
    f, sign = s["frequencies"], 1
    n = f.numel()
    turned = []
    for x in (s["q"], s["k"]):
        y = x.double().clone()
        for i in range(n):
            a, b = (2 * i, 2 * i + 1) if s["interleaved"] else (i, n + i)
            z = torch.polar(torch.full_like(s["positions"], sign, dtype=torch.float64) * s["magnitude"],
                            s["positions"].double() * f[i])[:, None] * torch.complex(x[..., a].double(), x[..., b].double())
            y[..., a], y[..., b] = z.real, z.imag
        turned.append(y)
    return tuple(turned)


def _exact_prompt(s):
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    starts, k_starts = s["offsets"].tolist(), s["k_offsets"].tolist()
    per = s["q"].shape[1] // s["k"].shape[1]
    for i in range(len(starts) - 1):
        n, m = starts[i + 1] - starts[i], k_starts[i + 1] - k_starts[i]
        for j in range(s["k"].shape[1]):
            k, v = (s[x][k_starts[i]:k_starts[i + 1], j].double().contiguous() for x in "kv")
            for g in range(j * per, (j + 1) * per):
                for first in range(0, n, 1024):
                    rows = min(1024, n - first)
                    part = slice(starts[i] + first, starts[i] + first + rows)
                    most = m - n + first + rows          # what the last of these sees
                    z = s["scale"] * torch.mm(s["q"][part, g].double().contiguous(), k[:most].t().contiguous())
                    z = z.tril(most - rows) + torch.full_like(z, -math.inf).triu(most - rows + 1)
                    out[part, g] = torch.mm(torch.softmax(z, 1), v[:most])
    return out


def _exact_tree(s):
    bits = torch.arange(256, device="cuda")
    e, f = (bits >> 3) & 15, (bits & 7).double()
    value = torch.where(e > 0, (1 + f / 8) * torch.exp2((e - 7).double()), f * 2.0 ** -9)
    value = torch.where(bits >= 128, -value, value)
    kc, vc, ke, ve = s["cache"]
    page = kc.shape[2]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    starts, tree = s["offsets"].tolist(), s["tree"].tolist()
    for i, length in enumerate(s["lengths"].tolist()):
        n = starts[i + 1] - starts[i]
        at = torch.arange(length, device="cuda")
        pg, row = s["table"][i].long()[at // page], at % page
        hidden = torch.zeros(n, length, dtype=torch.bool)
        for b in range(n):
            for j in range(n):
                hidden[b, length - n + j] = not (tree[starts[i] + b] >> j) & 1
        hidden = hidden.cuda()
        for j in range(kc.shape[1]):
            k = value[kc[pg, j, row].long()] * torch.exp2(ke[pg, j, row].double() - 127)[:, None]
            v = value[vc[pg, j, row // 16, :, row % 16].long()] * torch.exp2(ve[pg, j, row].double() - 127)[:, None]
            per = s["q"].shape[1] // kc.shape[1]
            for g in range(j * per, (j + 1) * per):
                z = s["scale"] * torch.mm(s["q"][starts[i]:starts[i + 1], g].double().contiguous(), k.t().contiguous())
                out[starts[i]:starts[i + 1], g] = torch.mm(torch.softmax(z.masked_fill(hidden, -math.inf), 1), v)
    return out


def _exact_place(s):
    """The two kinds of codes after a move or a copy, as 64-bit values."""
    held = [x.clone() for x in s["cache"][:2]]
    if s["op"] == "copy":
        for x, y in zip(held, s["cache"]):
            x.index_copy_(0, s["target"].long(), y.index_select(0, s["source"].long()))
    else:
        page = held[0].shape[2]
        at = s["source"] >= 0
        a, b = s["source"][at].long(), s["target"][at].long()
        for x, y, token in ((held[0], s["cache"][0], (0, 2, 1, 3)), (held[1], s["cache"][1], (0, 2, 4, 1, 3))):
            heads, dim = s["cache"][0].shape[1], s["cache"][0].shape[3]
            rows = y.permute(token).reshape(-1, heads, dim).clone()       # [slot][head][dim]
            rows[b] = rows[a]
            shape = [x.shape[i] for i in token]
            x.copy_(rows.view(shape).permute([token.index(i) for i in range(len(token))]))
            assert rows.shape[0] == x.shape[0] * page
    return tuple(x.view(torch.float8_e4m3fn).double() for x in held) + (None, None)


def exact(case, seed):
    s = prepare(case, seed)
    return {"rotary": _exact_rotary, "prompt": _exact_prompt, "tree": _exact_tree, "move": _exact_place,
            "copy": _exact_place}[case["op"]](s)
