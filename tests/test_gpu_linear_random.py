"""Random sizes through the 4-bit product and the gated projection: every tile, parts of the contraction and both ways of
taking a 4-bit weight, against 64-bit products on the GPU."""
import random

import pytest
import torch

import fp8_oracle as F8
import linear_oracle as O

pytestmark = pytest.mark.gpu


def _log(rng, low, high):
    return int(round(low * (high / low) ** rng.random()))


def _close(got, ref, off, dtype, what):
    got = got.detach().double()
    bound = O.rounded(ref, off, dtype)
    assert bool(torch.isfinite(got).all()), what
    past = float(((got - ref).abs() - bound).max())
    assert past <= 0, f"{what}: {past} past the bound"


def _product(a, w):
    return a @ w.t(), (a.shape[1] + 1) * O.SUM * (a.abs() @ w.abs().t())


@pytest.mark.parametrize("seed", range(24))
def test_linear(seed):
    from usaf_amd.moe import Q4Tensor
    from usaf_amd.q4 import q4_linear
    rng = random.Random(seed)
    dtype = rng.choice([torch.bfloat16, torch.float16])
    m, n, k = _log(rng, 1, 6000), _log(rng, 1, 6000), 128 * _log(rng, 1, 64)
    parts = [t.cuda() for t in O.codes(n, k, seed)]
    w = Q4Tensor(*parts, torch.Size((n, k)))
    w64 = w.dequantize(dtype).double()
    x = torch.randn(m, k, device="cuda", generator=torch.Generator("cuda").manual_seed(seed)).to(dtype).requires_grad_()
    y = q4_linear(x, w)
    _close(y, *_product(x.detach().double(), w64), dtype, f"out of {m} x {n} x {k}")
    dy = torch.randn(m, n, device="cuda", generator=torch.Generator("cuda").manual_seed(seed + 100)).to(dtype)
    y.backward(dy)
    _close(x.grad, *_product(dy.double(), w64.t()), dtype, f"dx of {m} x {n} x {k}")


@pytest.mark.parametrize("seed", range(24))
def test_gated(seed):
    from usaf_amd.gated import gated_linear
    from usaf_amd.moe import Q4Tensor
    rng = random.Random(seed)
    dtype, four, checkpoint = rng.choice([torch.bfloat16, torch.float16]), rng.random() < 0.5, rng.choice([None, "fp8"])
    m, inter = _log(rng, 1, 4000), _log(rng, 1, 3000)
    k = 128 * _log(rng, 1, 32) if four else _log(rng, 1, 4000)
    gen = torch.Generator("cuda").manual_seed(seed)
    if four:
        w = Q4Tensor(*[t.cuda() for t in O.codes(2 * inter, k, seed)], torch.Size((2 * inter, k)))
        w64 = w.dequantize(dtype).double()
    else:
        w = (torch.randn(2 * inter, k, device="cuda", generator=gen) * 0.05).to(dtype).requires_grad_()
        w64 = w.detach().double()
    x = torch.randn(m, k, device="cuda", generator=gen).to(dtype).requires_grad_()
    y = gated_linear(x, w, checkpoint=checkpoint)
    x64 = x.detach().double()
    (g, _), (u, _), (ref, off) = O.gated(x64, w64)
    _close(y, ref, off, dtype, f"act of {m} x {inter} x {k}")
    with torch.no_grad():
        _close(gated_linear(x, w), ref, off, dtype, f"act without a gradient of {m} x {inter} x {k}")
    # the gradients against the formula on gate and up as the 64-bit sums give them: what is kept is a rounding of
    # those (half a step of the type, of 4 significant bits with checkpoints), to which dG and dU react by less than 3 times its share
    dy = torch.randn(m, inter, device="cuda", generator=gen).to(dtype)
    y.backward(dy)
    (dg, _), (du, _) = O.gated_grads(dy.double(), g, u)
    dgu = torch.cat([dg, du], 1)
    share = 3 * (2.0 ** -4 if checkpoint else F8.half_step(dtype)) + 2 * F8.half_step(dtype)
    for got, want in ((x.grad, dgu @ w64), *(() if four else ((w.grad, dgu.t() @ x64),))):
        assert bool(torch.isfinite(got).all())
        assert float((got.double() - want).norm()) <= share * float(want.norm()) + 1e-6, f"{m} x {inter} x {k}"
