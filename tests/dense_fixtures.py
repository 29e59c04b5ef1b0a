"""The dense operators' definitions in 64 bits on the CPU, and their inputs
(not collected by pytest)."""
import numpy as np
import torch

HALF = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.float16, torch.bfloat16)}   # a rounding's most
U = 2.0 ** -24                                                                               # fp32's


def gen(seed):
    return torch.Generator().manual_seed(seed)


def near(got, want, tol, what):
    """|got - want| <= tol elementwise, NaN and infinities where `want` has them."""
    got, want, tol = got.detach().cpu().double(), want.double(), torch.as_tensor(tol, dtype=torch.float64)
    assert got.shape == want.shape, what
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN elsewhere"
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)]), f"{what}: infinities"
    over = ((got - want).abs() - tol.expand_as(want))[fine]
    assert over.numel() == 0 or over.max() <= 0, \
        f"{what}: off by {(got - want).abs()[fine].max():.3g}, {over.max():.3g} over its tolerance"


# ---------------------------------------------------------------- delta rule

def delta_inputs(seed, lens, key_heads, heads, dk, dv, dtype, normalize=True):
    r, n = gen(seed), sum(lens)
    q = torch.nn.functional.silu(torch.randn(n, key_heads, dk, generator=r)).to(dtype)
    k = torch.nn.functional.silu(torch.randn(n, key_heads, dk, generator=r))
    if not normalize:
        k = k / k.norm(dim=-1, keepdim=True).clamp(min=1e-3)
    v = torch.randn(n, heads, dv, generator=r).to(dtype)
    g = -0.3 * torch.rand(n, heads, generator=r) * torch.exp(torch.randn(heads, generator=r))
    beta = torch.rand(n, heads, generator=r)
    return q, k.to(dtype), v, g, beta


def delta(q, k, v, g, beta, state, lens, scale, normalize):
    """(o, final states): the recurrence, one token after another, from state
    [sequences][heads][dk][dv]."""
    q, k, v, g, beta = (x.double() for x in (q, k, v, g, beta))
    if normalize:
        q, k = (x / (x.square().sum(-1, keepdim=True) + 1e-6).sqrt() for x in (q, k))
    r = v.shape[1] // q.shape[1]
    q, k = q.repeat_interleave(r, 1), k.repeat_interleave(r, 1)
    o, final, t = torch.zeros_like(v), state.double().clone(), 0
    for i, n in enumerate(lens):
        s = final[i]
        for t in range(t, t + n):
            s = s * torch.exp(g[t])[:, None, None]
            u = beta[t][:, None] * (v[t] - (s * k[t][..., None]).sum(1))
            s = s + k[t][..., None] * u[:, None, :]
            o[t] = scale * (s * q[t][..., None]).sum(1)
        t += n > 0
        final[i] = s
    return o, final


def delta_tolerance(want, dtype, dk, longest, size):
    """One rounding of the output's type, and fp32 sums over dk terms whose
    errors the decaying, contracting state carries along but does not enlarge:
    a random walk of `longest` tokens, eight standard deviations of it, of
    values up to `size`."""
    return HALF[dtype] * want.abs() + 8 * U * (dk * (longest + 1)) ** 0.5 * size


# -------------------------------------------------------------- 4-bit weights

def q4_weights(seed, rows, cols, group, zeros, scale_type=torch.float16):
    r = gen(seed)
    codes = torch.randint(0, 256, (rows, cols // 2), dtype=torch.uint8, generator=r)
    scales = (0.02 * torch.randn(rows, cols // group, generator=r)).to(scale_type)
    z = torch.randint(0, 16, (rows, cols // group), dtype=torch.uint8, generator=r) if zeros else None
    return codes, scales, z


def q4(x, codes, scales, zeros):
    """(y, what its fp32 sums add up in magnitude)."""
    rows, groups = scales.shape
    w = torch.empty(rows, 2 * codes.shape[1], dtype=torch.float64)
    w[:, 0::2], w[:, 1::2] = (codes & 15).double(), (codes >> 4).double()
    g = w.shape[1] // groups
    z = (torch.full(scales.shape, 8.0) if zeros is None else zeros).double().repeat_interleave(g, 1)
    s = scales.double().repeat_interleave(g, 1)
    x = x.double()
    return x @ ((w - z) * s).T, x.abs() @ ((w + z) * s.abs()).T


# -------------------------------------------------------------- 8-bit cache

def e4m3():
    """The 256 values; NaN at 0x7f and 0xff."""
    b = np.arange(256)
    e, m = (b >> 3) & 15, (b & 7).astype(np.float64)
    v = np.where(e > 0, (1 + m / 8) * 2.0 ** (e - 7.0), m * 2.0 ** -9)
    v = np.where(b >= 128, -v, v)
    v[[0x7f, 0xff]] = np.nan
    return torch.from_numpy(v)


def held(x):
    """(values, codes, exponent bytes) of vectors along the last axis, by search
    among all codes: the nearest, at a tie the even one."""
    x = x.double()
    top = x.abs().amax(-1)
    bad = ~torch.isfinite(x).all(-1)
    e = torch.full(top.shape, -126.0, dtype=torch.float64)
    for p in range(-126, 121):
        e = torch.where(top * 2.0 ** -p > 448, torch.tensor(p + 1.0, dtype=torch.float64), e)
    table = e4m3()[:127]
    a = torch.where(bad[..., None], 0.0, x * torch.exp2(-e)[..., None])
    mag = a.abs()
    hi = torch.searchsorted(table.contiguous(), mag.contiguous()).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    dl, dh = mag - table[lo], table[hi] - mag
    code = torch.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    value = torch.where(a < 0, -table[code], table[code]) * torch.exp2(e)[..., None]
    value[bad] = torch.nan
    code = torch.where(torch.signbit(a), code + 128, code)
    exp = torch.where(bad, torch.tensor(255.0, dtype=torch.float64), e + 127)
    return value, code.to(torch.uint8), exp.to(torch.uint8)


def attend(q, k, v, lens, burst, scale):
    """k, v: a list of [tokens][heads][dim] per sequence."""
    q = q.double()
    o = torch.zeros_like(q)
    for i, n in enumerate(lens):
        r = q.shape[1] // k[i].shape[1]
        for b in range(burst):
            seen = n - burst + b + 1
            if seen <= 0:
                continue
            for h in range(q.shape[1]):
                p = torch.softmax(scale * (k[i][:seen, h // r].double() @ q[i * burst + b, h]), 0)
                o[i * burst + b, h] = p @ v[i][:seen, h // r].double()
    return o
