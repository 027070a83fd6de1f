"""The 8-bit block format and its product in 64 bits, on the CPU: the oracle of the
fp8 and few-token tests."""
import torch

BLOCK = 128


def half_step(dtype):
    """A rounding to dtype is off by at most this share of the value."""
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """... and by at most this near zero."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def e4m3(v):
    """Nearest e4m3 value (ties to even) of float64 values up to 448."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(v / step) * step


def exponent(amax):
    """Smallest integer e with amax 2^-e <= 448, in [-120, 120]."""
    m, e = torch.frexp(amax.double())  # amax = m 2^e, m in [1/2, 1); 448 = 7/8 2^9
    e = torch.where(m > 0.875, e - 8, e - 9)
    return torch.where(amax == 0, torch.full_like(e, -120), e.clamp(-120, 120))


def finite_amax(v, dims):
    return torch.where(torch.isfinite(v), v.abs(), torch.zeros_like(v)).amax(dims, keepdim=True)


def quantized_rows(x):
    """(values, E8M0 bytes [M, blocks]) of rows after quantization; values of non-finite entries NaN."""
    rows, cols = x.shape
    v = torch.nn.functional.pad(x.double(), (0, -cols % BLOCK)).view(rows, -1, BLOCK)
    e = exponent(finite_amax(v, -1))
    scale = torch.exp2(e.double())
    q = e4m3(torch.where(torch.isfinite(v), v, torch.full_like(v, float("nan"))) / scale) * scale
    return q.view(rows, -1)[:, :cols], (e + 127).squeeze(-1)


def quantized_weight(w):
    """The same for [.., R, C] in blocks of 128 x 128."""
    *lead, r, c = w.shape
    v = torch.nn.functional.pad(w.double(), (0, -c % BLOCK, 0, -r % BLOCK))
    v = v.view(*lead, v.shape[-2] // BLOCK, BLOCK, v.shape[-1] // BLOCK, BLOCK)
    e = exponent(finite_amax(v, (-3, -1)))
    scale = torch.exp2(e.double())
    q = e4m3(torch.where(torch.isfinite(v), v, torch.full_like(v, float("nan"))) / scale) * scale
    q = q.reshape(*lead, v.shape[-4] * BLOCK, v.shape[-2] * BLOCK)[..., :r, :c]
    return q, (e + 127).squeeze(-1).squeeze(-2)


def values(q, s, shape):
    """Values of uint8 codes and E8M0 bytes."""
    *lead, r, c = shape
    scale = torch.exp2(s.double() - 127).repeat_interleave(BLOCK, -1).repeat_interleave(BLOCK, -2)
    return (q.view(torch.float8_e4m3fn).double() * scale[..., :r, :])[..., :c]


def product_bound(a, w, ref, dtype):
    """How far a product of values a [M, K], w [N, K] on the 8-bit matrix instruction, rounded to dtype, may be from ref.

    The output is off by at most half a step.  Every addition to the fp32 accumulator is off by at most 2^-23 of
    the magnitudes so far (a whole step: it may cut).  Within one instruction (64 products) the products are
    aligned to the largest and cut: one of 2^-13 of it arrives whole, one of 2^-14 not at all (measured
    with powers of two beside a pair that cancels), so each of the 64 loses less than 2^-13 of the largest, together less than
    2^-7 max|a| max|w| of those 64.  (The instruction's measured error on normal data is 1.5e-5 of the result, rms.)"""
    mags = a.abs() @ w.abs().t()
    pad = (0, -a.shape[1] % 64)
    top = [torch.nn.functional.pad(v.abs(), pad).view(v.shape[0], -1, 64).amax(-1) for v in (a, w)]
    cut = 2.0 ** -7 * (top[0] @ top[1].t())
    return ref.abs() * half_step(dtype) + tiny(dtype) + ((a.shape[1] + 1) * 2.0 ** -23 * mags + cut) * (1 + half_step(dtype))


def wide_bound(a, w, ref, dtype):
    """As product_bound for the 16-bit instruction, which cuts nothing: the output's half step and the fp32 sum's steps."""
    mags = a.abs() @ w.abs().t()
    return ref.abs() * half_step(dtype) + tiny(dtype) + (a.shape[1] + 1) * 2.0 ** -23 * mags * (1 + half_step(dtype))
