"""The dense operators that are timed, through their public entry points.

The expert engine computes the experts of a hybrid model whose other layers mix
tokens by a gated delta rule (three of four) or by attention. These are the
operators of that dense part, for the same card and stream:

  delta   fronk_amd.dense.delta_rule: the gated delta rule over ragged
          sequences, from one token (decode) to a prompt, state in and out;
  q4      fronk_amd.dense.q4_product: y = x W^T with 4-bit weights, one scale
          (and, where given, one zero point) per group of a row;
  write   fronk_amd.dense.kv_append and kv_read: a paged cache held in 8 bits
          (e4m3 codes, one power of two per token and head), written and read;
  attend  fronk_amd.dense.kv_attend: bursts of 1 to 8 tokens attending to it.

`run` in its plain form computes the same in 32 bits from elementary torch
operations. The layouts of the 4-bit weights and of the cache are the public
ones that fronk_amd.dense documents, so both forms take the same state.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
CHUNK = 64


def _delta(name, seqs, tokens, key_heads, heads, dk, dv, dtype, normalize=True, ragged=False, initial=True):
    return {"name": name, "op": "delta", "seqs": seqs, "tokens": tokens, "key_heads": key_heads, "heads": heads,
            "dk": dk, "dv": dv, "dtype": dtype, "normalize": normalize, "ragged": ragged, "initial": initial}


def _q4(name, tokens, cols, rows, group, dtype, zeros=False):
    return {"name": name, "op": "q4", "tokens": tokens, "cols": cols, "rows": rows, "group": group, "dtype": dtype,
            "zeros": zeros}


def _write(name, tokens, kv_heads, dim, page, dtype):
    return {"name": name, "op": "write", "tokens": tokens, "kv_heads": kv_heads, "dim": dim, "page": page,
            "dtype": dtype}


def _attend(name, seqs, burst, context, heads, kv_heads, dim, page, dtype, ragged=False):
    return {"name": name, "op": "attend", "seqs": seqs, "burst": burst, "context": context, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype, "ragged": ragged}


def listed():
    return [
        # One user's next token: the smallest state there is to move.
        _delta("delta_token", 1, 1, 16, 32, 128, 128, "bf16"),
        # A serving batch, each stream with one to four tokens to verify.
        _delta("delta_batch", 64, 4, 16, 32, 128, 128, "bf16", ragged=True),
        # A few prompts of unequal length, other head sizes, 32-bit activations.
        _delta("delta_ragged", 5, 701, 3, 9, 64, 80, "f32", ragged=True),
        # The longest prefill chunk the expert engine takes, from an empty state.
        _delta("delta_prompt", 1, 4096, 16, 32, 128, 128, "bf16", initial=False),
        # A projection of one token, the runtime's own hidden size.
        _q4("q4_token", 1, 2560, 2560, 64, "bf16"),
        # The vocabulary's projection of one token, the largest read there is.
        _q4("q4_vocabulary", 1, 4096, 65536, 128, "bf16"),
        # A burst with 32-bit activations, zero points, rows that fill no tile.
        _q4("q4_burst", 7, 2592, 4099, 32, "f32", zeros=True),
        # A prefill chunk's projection.
        _q4("q4_chunk", 512, 4096, 8192, 128, "bf16"),
        # One token of one stream into the cache.
        _write("write_token", 1, 2, 256, 64, "bf16"),
        # A prefill chunk into the cache.
        _write("write_chunk", 4096, 2, 256, 64, "bf16"),
        # One stream over a long context.
        _attend("attend_long", 1, 1, 131072, 16, 2, 256, 64, "bf16"),
        # A serving batch with speculative tokens over unequal contexts.
        _attend("attend_batch", 32, 4, 8192, 16, 2, 128, 32, "bf16", ragged=True),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["delta", "delta", "q4", "q4", "write", "attend", "attend"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "delta":
        key_heads = rng.choice([1, 2, 3, 4, 5, 8, 16])
        heads = key_heads * rng.choice([1, 2, 2, 3, 4])
        heads = heads if heads <= 32 else 2 * key_heads
        dk, dv = rng.choice([64, 128, 128, 256]), 16 * rng.randint(2, 8)
        if dk == 256:
            heads, key_heads = (heads // key_heads) * min(key_heads, 4), min(key_heads, 4)
        if rng.random() < 0.5:
            seqs, tokens = _log_int(rng, 1, 64), rng.randint(1, 8)
        else:
            seqs = rng.randint(1, 6)
            tokens = _log_int(rng, 9, 4096 // seqs)
        c = _delta("", seqs, tokens, key_heads, heads, dk, dv, dtype, rng.random() < 0.7, rng.random() < 0.5,
                   rng.random() < 0.7)
    elif op == "q4":
        group = rng.choice([32, 64, 128])
        cols = group * max(1, _log_int(rng, 256, 8192) // group)
        tokens = rng.randint(1, 8) if rng.random() < 0.6 else _log_int(rng, 9, 512)
        rows = _log_int(rng, 1, 65536 if tokens == 1 else 16384)
        rows = min(rows, max(1, 512 * 4096 * 8192 // (tokens * cols)), 65536 * 4096 // cols)
        c = _q4("", tokens, cols, rows, group, dtype, rng.random() < 0.5)
    elif op == "write":
        c = _write("", _log_int(rng, 1, 4096), rng.choice([1, 2, 3, 4, 8]), rng.choice([64, 128, 256]),
                   rng.choice([16, 32, 64, 128]), dtype)
        c["tokens"] = min(c["tokens"], 4096 * 512 // (c["kv_heads"] * c["dim"]))
    else:
        kv_heads = rng.choice([1, 2, 2, 4, 8])
        dim = rng.choice([64, 128, 256])
        seqs = _log_int(rng, 1, 64)
        most = 131072 * 512 // (seqs * kv_heads * dim)
        c = _attend("", seqs, rng.choice([1, 1, 2, 3, 5, 8]), _log_int(rng, 8, min(most, 131072)),
                    kv_heads * rng.choice([1, 2, 3, 4, 7, 8]), kv_heads, dim, rng.choice([16, 32, 64, 128]), dtype,
                    rng.random() < 0.6)
    del c["name"]
    return c


# ------------------------------------------------------------------ inputs

def _lengths(case):
    """The sequences' lengths, from the case alone: all of them `tokens` (delta)
    or `context` (attend), or spread evenly from one up to it."""
    top = case["tokens"] if case["op"] == "delta" else case["context"]
    low = 1 if case["op"] == "delta" else min(top, case["burst"])
    n = case["seqs"]
    if not case["ragged"] or n == 1:
        return [top] * n
    return [low + ((7 * i + 3) % n) * (top - low) // (n - 1) for i in range(n)]


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _prepare_delta(case, rand):
    lens, dt = _lengths(case), TYPES[case["dtype"]]
    total, hk, h, dk, dv = sum(lens), case["key_heads"], case["heads"], case["dk"], case["dv"]
    # q, k and v as the layer's convolution leaves them: one row per token,
    # SiLU of a normal value, so that keys lean to one side.
    row = torch.nn.functional.silu(rand(total, hk * dk * 2 + h * dv) * 1.5).to(dt)
    q = row[:, :hk * dk].unflatten(1, (hk, dk))
    k = row[:, hk * dk:2 * hk * dk].unflatten(1, (hk, dk))
    v = row[:, 2 * hk * dk:].unflatten(1, (h, dv))
    if not case["normalize"]:
        k = (k.float() / (k.float().square().sum(-1, keepdim=True) + 1e-6).sqrt()).to(dt)
    g = -torch.exp(rand(h)) * torch.nn.functional.softplus(rand(total, h) - 2)
    state = 0.3 * rand(case["seqs"] + 1, h, dk, dv)
    starts = [sum(lens[:i]) for i in range(len(lens) + 1)]
    return {"q": q, "k": k, "v": v, "g": g, "beta": torch.sigmoid(rand(total, h)), "state": state,
            "offsets": _ints(starts), "slots": _ints([(i + 1) % (case["seqs"] + 1) for i in range(case["seqs"])]),
            "max_tokens": max(lens), "scale": dk ** -0.5, "normalize": case["normalize"], "initial": case["initial"]}


def _prepare_q4(case, rand):
    n, k, g = case["rows"], case["cols"], case["group"]
    codes = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device="cuda", generator=rand.generator)
    scales = (0.01 * (0.2 + torch.rand(n, k // g, device="cuda", generator=rand.generator))).to(torch.float16)
    zeros = torch.randint(5, 11, (n, k // g), dtype=torch.uint8, device="cuda", generator=rand.generator)
    x = rand(case["tokens"], k)
    x[:, torch.randint(0, k, (4,), device="cuda", generator=rand.generator)] *= 8.0
    return {"x": x.to(TYPES[case["dtype"]]), "codes": codes, "scales": scales, "zeros": zeros if case["zeros"] else None}


def _empty_cache(pages, heads, page, dim):
    """The cache's four arrays (fronk_amd.dense.KVCache): K codes by token, V
    codes by blocks of 16 tokens, and the two exponents."""
    kw = {"dtype": torch.uint8, "device": "cuda"}
    return (torch.zeros(pages, heads, page, dim, **kw), torch.zeros(pages, heads, page // 16, dim, 16, **kw),
            torch.zeros(pages, heads, page, **kw), torch.zeros(pages, heads, page, **kw))


def _prepare_write(case, rand):
    t, h, d, p = case["tokens"], case["kv_heads"], case["dim"], case["page"]
    pages = (t + p - 1) // p + 1
    kv = rand(t, 2 * h * d) * torch.exp(rand(t, 1))
    kv = kv.to(TYPES[case["dtype"]])
    order = torch.randperm(pages, device="cuda", generator=rand.generator)
    at = torch.arange(t, device="cuda") + p // 2      # the stream goes on in the middle of a page
    slots = (order[at // p] * p + at % p).to(torch.int32)
    return {"k": kv[:, :h * d].unflatten(1, (h, d)), "v": kv[:, h * d:].unflatten(1, (h, d)), "slots": slots,
            "cache": _empty_cache(pages, h, p, d)}


def _prepare_attend(case, rand):
    lens, p, h, d = _lengths(case), case["page"], case["kv_heads"], case["dim"]
    per = (max(lens) + p - 1) // p
    pages = case["seqs"] * per
    kc, vc, ke, ve = _empty_cache(pages, h, p, d)
    # Codes of normal values at a scale that puts their largest near 448, and
    # the exponents that bring them back to about one.
    for codes in (kc, vc):
        flat = codes.view(-1)
        for i in range(0, flat.numel(), 1 << 26):
            part = flat[i:i + (1 << 26)]
            part.copy_((100 * rand(part.numel())).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8))
    for e in (ke, ve):
        e.copy_(torch.randint(119, 122, e.shape, device="cuda", generator=rand.generator))
    table = torch.randperm(pages, device="cuda", generator=rand.generator).to(torch.int32).view(case["seqs"], per)
    q = rand(case["seqs"] * case["burst"], case["heads"], d).to(TYPES[case["dtype"]])
    return {"q": q, "cache": (kc, vc, ke, ve), "table": table, "lengths": _ints(lens), "context": max(lens),
            "scale": 2.0 * d ** -0.5}


class _Rand:
    """Normal values on the GPU from one seeded generator."""

    def __init__(self, seed):
        self.generator = torch.Generator(device="cuda")
        self.generator.manual_seed(seed)

    def __call__(self, *shape):
        return torch.randn(*shape, device="cuda", generator=self.generator)


def prepare(case, seed):
    make = {"delta": _prepare_delta, "q4": _prepare_q4, "write": _prepare_write, "attend": _prepare_attend}
    return {"op": case["op"], **make[case["op"]](case, _Rand(seed))}


# ------------------------------------------------------------------ one pass

def run(state):
    s = dict(state)
    op = s.pop("op")
    if own:
        from fronk_amd import dense
        if op == "delta":
            o = dense.delta_rule(s["q"], s["k"], s["v"], s["g"], s["beta"], s["state"] if s["initial"] else None,
                                 s["state"], scale=s["scale"], offsets=s["offsets"], slots=s["slots"],
                                 max_tokens=s["max_tokens"], normalize=s["normalize"])
            return o, s["state"]
        if op == "q4":
            return dense.q4_product(s["x"], s["codes"], s["scales"], s["zeros"])
        if op == "write":
            dense.kv_append(s["cache"], s["k"], s["v"], s["slots"])
            return dense.kv_read(s["cache"], s["slots"], s["k"].dtype)
        return dense.kv_attend(s["cache"], s["q"], s["table"], s["lengths"], scale=s["scale"],
                               max_context=s["context"])
    return {"delta": _plain_delta, "q4": _plain_q4, "write": _plain_write, "attend": _plain_attend}[op](**s)


def _plain_delta(q, k, v, g, beta, state, offsets, slots, max_tokens, scale, normalize, initial):
    """Chunks of 64 tokens: within one, the updates' values solve a lower
    triangular system; from one to the next goes the state."""
    dtype, r = v.dtype, v.shape[1] // q.shape[1]
    seqs, c = slots.shape[0], min(CHUNK, max_tokens)
    n = (max_tokens + c - 1) // c
    at = offsets[:-1, None].long() + torch.arange(n * c, device=q.device)
    live = at < offsets[1:, None]
    at = torch.where(live, at, 0)

    def rows(x, repeat=1):   # [token][head][...] -> [sequence][head][chunk][row][...]
        x = x.float()[at] * live.view(live.shape + (1,) * (x.dim() - 1))
        return x.repeat_interleave(repeat, 2).unflatten(1, (n, c)).movedim(3, 1)

    def unit(x):
        return x * torch.rsqrt(x.square().sum(-1, keepdim=True) + 1e-6) if normalize else x

    q, k, v = unit(rows(q, r)) * scale, unit(rows(k, r)), rows(v)
    total, b = torch.cumsum(rows(g), -1), rows(beta)
    i = torch.arange(c, device=q.device)
    decay = torch.exp(torch.where(i[:, None] >= i, total[..., :, None] - total[..., None, :], -math.inf))
    kt = k.transpose(-1, -2).contiguous()
    a = b[..., None] * (k @ kt) * decay * (i[:, None] > i)
    inverse = torch.eye(c, device=q.device).expand_as(a).clone()
    for row in range(1, c):
        inverse[..., row, :row] = -(a[..., row, None, :row] @ inverse[..., :row, :row])[..., 0, :]
    u = inverse @ (b[..., None] * v)
    w = inverse @ (b[..., None] * torch.exp(total)[..., None] * k)
    within = (q @ kt) * decay
    across = q * torch.exp(total)[..., None]
    last = total[..., -1:]
    kt = kt * torch.exp(last - total)[..., None, :]
    s = state[slots.long()] if initial else torch.zeros_like(state[1:])
    out = torch.zeros_like(u)
    for j in range(n):
        new = u[:, :, j] - w[:, :, j] @ s
        out[:, :, j] = across[:, :, j] @ s + within[:, :, j] @ new
        s = s * torch.exp(last[:, :, j])[..., None] + kt[:, :, j] @ new
    state[slots.long()] = s
    out = out.movedim(1, 3).flatten(1, 2)
    return out[live].to(dtype), state


def _plain_q4(x, codes, scales, zeros):
    n, groups = scales.shape
    w = torch.stack([codes & 15, codes >> 4], dim=2).view(n, groups, -1).float()
    w = (w - (8.0 if zeros is None else zeros.float()[..., None])) * scales.float()[..., None]
    return (x.float() @ w.view(n, -1).T).to(x.dtype)


def _quantize(x):
    """(codes as e4m3, exponents): the smallest power of two that brings the
    largest of a token's head within 448."""
    x = x.float()
    top = x.abs().amax(-1)
    m, e = torch.frexp(top)
    e = torch.where(top > 0, e - 9 + (m > 0.875).int(), -126).clamp(-126, 127)
    return torch.ldexp(x, -e[..., None]).to(torch.float8_e4m3fn).view(torch.uint8), (e + 127).to(torch.uint8)


def _values(codes, exponents):
    return torch.ldexp(codes.view(torch.float8_e4m3fn).float(), exponents.int()[..., None] - 127)


def _plain_write(k, v, slots, cache):
    kc, vc, ke, ve = cache
    page, at = slots.long() // kc.shape[2], slots.long() % kc.shape[2]
    (kq, kx), (vq, vx) = _quantize(k), _quantize(v)
    kc[page, :, at], ke[page, :, at] = kq, kx
    vc[page, :, at // 16, :, at % 16], ve[page, :, at] = vq, vx
    return (_values(kc[page, :, at], ke[page, :, at]).to(k.dtype),
            _values(vc[page, :, at // 16, :, at % 16], ve[page, :, at]).to(v.dtype))


def _plain_attend(q, cache, table, lengths, context, scale):
    kc, vc, ke, ve = cache
    seqs, h, d = table.shape[0], kc.shape[1], q.shape[2]
    burst, r = q.shape[0] // seqs, q.shape[1] // h
    t = table.long()
    k = _values(kc[t], ke[t]).transpose(1, 2).flatten(2, 3)[:, :, :context]       # [sequence][head][token][d]
    v = vc[t].transpose(-1, -2).flatten(3, 4)
    v = _values(v, ve[t]).transpose(1, 2).flatten(2, 3)[:, :, :context]
    qs = q.float().view(seqs, burst, h, r, d).permute(0, 2, 1, 3, 4).reshape(seqs, h, burst * r, d)
    p = (qs @ k.transpose(-1, -2)) * scale
    last = lengths[:, None].long() - burst + torch.arange(burst, device=q.device)
    seen = torch.arange(context, device=q.device) <= last[..., None]
    seen = seen[:, None, :, None, :].expand(seqs, 1, burst, r, context).reshape(seqs, 1, burst * r, context)
    p = torch.where(seen, p, -math.inf)
    top = p.amax(-1, keepdim=True)
    p = torch.exp(p - torch.where(top > -math.inf, top, 0.0))
    o = (p @ v) / p.sum(-1, keepdim=True)
    return o.view(seqs, h, burst, r, d).permute(0, 2, 1, 3, 4).reshape(q.shape).to(q.dtype)


def work(case):
    size = SIZE[case["dtype"]]
    if case["op"] == "delta":
        t, h, dk, dv = sum(_lengths(case)), case["heads"], case["dk"], case["dv"]
        states = 4 * case["seqs"] * h * dk * dv
        return {"bytes": t * (size * (2 * case["key_heads"] * dk + 2 * h * dv) + 8 * h)
                + states * (2 if case["initial"] else 1), "flops": 7 * t * h * dk * dv}
    if case["op"] == "q4":
        t, k, n = case["tokens"], case["cols"], case["rows"]
        weights = n * k // 2 + n * (k // case["group"]) * (3 if case["zeros"] else 2)
        return {"bytes": weights + size * t * (k + n), "flops": 2 * t * k * n}
    if case["op"] == "write":
        values = 2 * case["tokens"] * case["kv_heads"] * case["dim"]
        # read, written as codes, read again, written as values
        return {"bytes": values * (2 * size + 2) + 4 * case["tokens"] * case["kv_heads"], "flops": 3 * values}
    tokens, d = sum(_lengths(case)), case["dim"]
    return {"bytes": tokens * case["kv_heads"] * (2 * d + 2) + 2 * size * case["seqs"] * case["burst"] * case["heads"] * d,
            "flops": 4 * tokens * case["burst"] * case["heads"] * d}


# ------------------------------------------------------- the result in 64 bits

def _fold(s, x):
    """sum over d of s[..., d, c] * x[..., d]"""
    return (s * x[..., None]).sum(-2)


def _exact_delta(s):
    """The recurrence, one token after another."""
    q, k, v, g, beta = (s[n].double() for n in ("q", "k", "v", "g", "beta"))
    if s["normalize"]:
        q, k = (x / (x.square().sum(-1, keepdim=True) + 1e-6).sqrt() for x in (q, k))
    r = v.shape[1] // q.shape[1]
    starts, slots = s["offsets"].tolist(), s["slots"].long()
    state = s["state"].double()
    live = state[slots] if s["initial"] else torch.zeros_like(state[slots])
    out = torch.zeros_like(v)
    for t in range(s["max_tokens"]):
        on = [i for i in range(len(starts) - 1) if starts[i] + t < starts[i + 1]]
        at = torch.tensor([starts[i] + t for i in on], device=q.device)
        w = slice(None) if len(on) == len(starts) - 1 else torch.tensor(on, device=q.device)
        kt, qt = k[at].repeat_interleave(r, 1), q[at].repeat_interleave(r, 1)
        now = live[w] * torch.exp(g[at])[..., None, None]
        u = beta[at][..., None] * (v[at] - _fold(now, kt))
        now = now + kt[..., None] * u[..., None, :]
        out[at] = s["scale"] * _fold(now, qt)
        live[w] = now
    state[slots] = live
    return out, state


def _exact_q4(s):
    codes, scales = s["codes"].long(), s["scales"].double()
    n, groups = scales.shape
    width = 2 * codes.shape[1] // groups
    x = s["x"].double()
    y = torch.empty(x.shape[0], n, dtype=torch.float64, device=x.device)
    for i in range(0, n, 4096):
        part = codes[i:i + 4096]
        w = torch.empty(part.shape[0], 2 * part.shape[1], dtype=torch.float64, device=x.device)
        w[:, 0::2], w[:, 1::2] = part % 16, part // 16
        zero = torch.full_like(scales, 8) if s["zeros"] is None else s["zeros"].double()
        w -= zero[i:i + 4096].repeat_interleave(width, 1)
        w *= scales[i:i + 4096].repeat_interleave(width, 1)
        y[:, i:i + 4096] = x @ w.T
    return y


def _exact_write(s):
    def held(x):
        x = x.double()
        top = x.abs().amax(-1, keepdim=True)
        e = torch.ceil(torch.log2(torch.where(top > 0, top / 448, torch.ones_like(top))))
        e = torch.where(top * torch.exp2(-e) > 448, e + 1, e)          # log2 may round to either side of a power
        e = torch.where(top * torch.exp2(1 - e) <= 448, e - 1, e)
        e = torch.where(top > 0, e, torch.zeros_like(e)).clamp(-126, 127)
        a = x * torch.exp2(-e)
        grid = torch.exp2(torch.floor(torch.log2(a.abs().clamp(min=2.0 ** -6))) - 3)
        return torch.round(a / grid) * grid * torch.exp2(e)
    return held(s["k"]), held(s["v"])


def _exact_attend(s):
    bits = torch.arange(256, device="cuda")
    e, m = (bits >> 3) & 15, (bits & 7).double()
    table = torch.where(e > 0, (1 + m / 8) * torch.exp2((e - 7).double()), m * 2.0 ** -9)
    table = torch.where(bits >= 128, -table, table)
    kc, vc, ke, ve = s["cache"]
    q, burst = s["q"].double(), s["q"].shape[0] // s["table"].shape[0]
    page, d = kc.shape[2], kc.shape[3]
    out = torch.empty_like(q)
    for i, length in enumerate(s["lengths"].tolist()):
        at = torch.arange(length, device="cuda")
        pg, row = s["table"][i].long()[at // page], at % page
        for j in range(kc.shape[1]):
            k = table[kc[pg, j, row].long()] * torch.exp2(ke[pg, j, row].double() - 127)[:, None]
            v = table[vc[pg, j, row // 16, :, row % 16].long()] * torch.exp2(ve[pg, j, row].double() - 127)[:, None]
            r = q.shape[1] // kc.shape[1]
            for b in range(burst):
                seen = length - burst + b + 1
                z = (k[:seen] @ q[i * burst + b, j * r:(j + 1) * r].T) * s["scale"]
                out[i * burst + b, j * r:(j + 1) * r] = torch.softmax(z, 0).T @ v[:seen]
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"delta": _exact_delta, "q4": _exact_q4, "write": _exact_write, "attend": _exact_attend}[case["op"]](s)
