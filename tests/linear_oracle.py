"""The 4-bit product and the gated projection in 64 bits, on the CPU, with how far a
kernel may be off: the oracle of their tests."""
import torch

from fp8_oracle import half_step, tiny

SUM = 2.0 ** -23  # every addition to an fp32 accumulator is off by at most this share of the magnitudes so far (it may cut)


def codes(rows, k, seed=0, scale=0.01):
    """(codes int8 [groups, 64], fp16 scales, fp16 zeros) of a random 4-bit weight [rows, k]: some groups flat, some of
    scales and zeros at the type's low end."""
    gen = torch.Generator().manual_seed(seed)
    n = rows * k // 128
    q = torch.randint(0, 256, (n, 64), dtype=torch.uint8, generator=gen).view(torch.int8)
    s = scale * (0.3 + torch.rand(n, generator=gen))
    z = -7.5 * s * (0.8 + 0.4 * torch.rand(n, generator=gen))
    s[::7] = 2.0 ** -20
    z[3::11] = 2.0 ** -22
    return q, s.half(), z.half()


def weight(q, s, z, rows, k, dtype):
    """float64 values of the codec in dtype: fp16(fp16(code * scale) + zero), then dtype (all exact roundings of torch's CPU)."""
    b = q.view(torch.uint8)
    c = torch.stack([b & 15, b >> 4], dim=-1).view(-1, 128).float()
    v = ((c * s.float()[:, None]).half().float() + z.float()[:, None]).half()
    return v.to(dtype).double().view(rows, k)


def product(a, w):
    """(a w^T, how far the fp32 sum may be from it) of float64 values."""
    ref = a @ w.t()
    return ref, (a.shape[1] + 1) * SUM * (a.abs() @ w.abs().t())


def rounded(ref, off, dtype):
    """How far dtype(value) may be from ref, for a value that is within off of it."""
    return off + (ref.abs() + off) * half_step(dtype) + tiny(dtype)


def gated(x, w):
    """gate, up, act in 64 bits and how far each may be off before its rounding.

    act = silu(g) u: |d silu / dg| <= 1.1.  The kernel's silu is g / (1 + 2^(-g log2 e)) with the hardware's exp2 and
    reciprocal (one unit each, 2^-23) on an argument rounded twice (2^-24 |g| each, times ln 2 log2 e = 1), one addition and two
    products: (2 |g| + 8) 2^-23 covers them."""
    inter = w.shape[0] // 2
    g, off_g = product(x, w[:inter])
    u, off_u = product(x, w[inter:])
    silu = g * torch.sigmoid(g)
    act = silu * u
    off = 1.1 * off_g * (u.abs() + off_u) + silu.abs() * off_u + act.abs() * (2 * g.abs() + 8) * SUM
    return (g, off_g), (u, off_u), (act, off)


def gated_grads(dact, g, u):
    """dG, dU of kept values in 64 bits and how far the fp32 formulas may be off.

    s as above; 1 + g (1 - s) adds terms of 1 and |g| (1 - s) <= |g|: each of its roundings is at most (1 + |g|) 2^-23, and the
    error of s, (2 |g| + 8) 2^-23 s, enters it times |g|."""
    s = torch.sigmoid(g)
    dg, du = dact * u * s * (1 + g * (1 - s)), dact * g * s
    rel = (2 * g.abs() + 8) * SUM
    off_g = (dact * u * s).abs() * (rel * (1 + g.abs()) * 2 + 4 * SUM * (1 + g.abs()))
    return (dg, off_g), (du, du.abs() * (rel + 2 * SUM))


def within(got, ref, bound, what=""):
    got = got.detach().double().cpu()
    assert got.shape == ref.shape, (got.shape, ref.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), what
    fine = torch.isfinite(ref)
    off = ((got - ref).abs() - bound)[fine]
    assert off.numel() == 0 or float(off.max()) <= 0, f"{what}: {float(off.max())} past the bound"


def rms_off(got, ref):
    got = got.detach().double().cpu()
    return float((got - ref).pow(2).mean().sqrt() / ref.pow(2).mean().sqrt())
