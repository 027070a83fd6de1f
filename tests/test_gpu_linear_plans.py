"""Every kernel of the 4-bit product and the gated projection, forward and backward, against 64-bit products on the GPU, at
sizes that are known to take it."""
import pytest
import torch

import fp8_oracle as F8
import linear_oracle as O
import linear_plans as P
from usaf_amd import gated as G
from usaf_amd.moe import Q4Tensor
from usaf_amd.q4 import q4_linear

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]


def _within(got, ref, bound, what):
    assert got.shape == ref.shape and bool(torch.isfinite(got).all()), what
    past = float(((got.detach().double() - ref).abs() - bound).max())
    assert past <= 0, f"{what}: {past} past the bound"


def _close(got, ref, off, dtype, what):
    """Within off and a rounding of ref everywhere, and on the whole no further than one and a half roundings: those of dG
    and dU, a third of half a step squared each on the whole, and of the result add up like random ones."""
    _within(got, ref, O.rounded(ref, off, dtype), what)
    if ref.numel() >= 4096:
        off = float((got.detach().double() - ref).norm() / ref.norm())
        assert off <= 1.5 * F8.half_step(dtype), f"{what}: {off} of the whole"


def _rand(*shape, seed, dtype, scale=1.0):
    return (torch.randn(*shape, device="cuda", generator=torch.Generator("cuda").manual_seed(seed)) * scale).to(dtype)


def _kept(x, w, checkpoint, g, off_g, u, off_u, dtype):
    """Gate and up as a forward keeps them for its backward, which are the oracle's up to their rounding."""
    inter = g.shape[1]
    with torch.no_grad():
        act, kept, scales = G._forward(x.detach(), w if isinstance(w, Q4Tensor) else w.detach(), checkpoint, True)
    if checkpoint is None:
        values = kept.double()
    else:
        s = torch.exp2(scales.double() - 127)
        values = kept.view(torch.float8_e4m3fn).double() * s.repeat_interleave(128, -1)
        assert not values[:, :, inter:].any()  # codes behind the last column are zeros
    values = [values[:, i, :inter] for i in range(2)]
    for i, (ref, off) in enumerate(((g, off_g), (u, off_u))):
        what = ("gate", "up")[i]
        if checkpoint is None:
            _within(values[i], ref, O.rounded(ref, off, dtype), what)
            continue
        # the scale is the oracle's for a largest magnitude within the sum's error; a code is at most half a step off
        low, high = (torch.nn.functional.pad((ref.abs() + sign * off).clamp_min(0), (0, -inter % 128)).view(len(ref), -1, 128)
                     .amax(-1).cpu() for sign in (-1, 1))
        e = torch.log2(s[:, i]).long().cpu()
        assert bool((F8.exponent(low) <= e).all()) and bool((e <= F8.exponent(high)).all()), what
        step = s[:, i].repeat_interleave(128, -1)[:, :inter]
        _within(values[i], ref, torch.maximum((ref.abs() + off) * 2.0 ** -4, step * 2.0 ** -10) * (1 + 2.0 ** -20) + off, what)
    return act, values


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda d: str(d).replace("torch.", ""))
@pytest.mark.parametrize("case", P.CASES, ids=lambda c: "-".join(map(str, c[:5])))
def test_kernels(case, dtype):
    call, m, n, k, checkpoint, plans = case
    assert P.plans(*case[:5]) == plans
    rows = n if call == "q4" else 2 * n
    x = _rand(m, k, seed=1, dtype=dtype).requires_grad_()
    if call == "gated16":
        w = _rand(rows, k, seed=2, dtype=dtype, scale=1.5 * k ** -0.5).requires_grad_()
        w64 = w.detach().double()
    else:
        parts = O.codes(rows, k, m + n, 0.3 * k ** -0.5)
        w = Q4Tensor(*(t.cuda() for t in parts), torch.Size((rows, k)))
        w64 = O.weight(*parts, rows, k, dtype).cuda()
    x64, dy = x.detach().double(), _rand(m, n, seed=3, dtype=dtype)
    if call == "q4":
        y = q4_linear(x, w)
        _close(y, *O.product(x64, w64), dtype, "out")
        y.backward(dy)
        _close(x.grad, *O.product(dy.double(), w64.t()), dtype, "dx")
        return
    (g, off_g), (u, off_u), (ref, off) = O.gated(x64, w64)
    y = G.gated_linear(x, w, checkpoint)
    _close(y, ref, off, dtype, "act")
    with torch.no_grad():
        _close(G.gated_linear(x, w), ref, off, dtype, "act without a gradient")
    again, (g, u) = _kept(x, w, checkpoint, g, off_g, u, off_u, dtype)
    assert torch.equal(again, y)
    y.backward(dy)
    (dg, od_g), (du, od_u) = O.gated_grads(dy.double(), g, u)
    dgu, od = torch.cat([dg, du], 1), torch.cat([od_g, od_u], 1)
    od = O.rounded(dgu, od, dtype)
    ref, off = O.product(dgu, w64.t())
    _close(x.grad, ref, off + od @ w64.abs(), dtype, "dx")
    if call == "gated16":
        ref, off = O.product(dgu.t(), x64.t())
        _close(w.grad, ref, off + od.t() @ x64.abs(), dtype, "dw")
