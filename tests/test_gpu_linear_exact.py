"""Products whose every rounding is known: outputs equal to the last bit, so each value of both operands is in its place."""
import pytest
import torch

import linear_oracle as O
import linear_plans as P
from usaf_amd.gated import gated_linear
from usaf_amd.moe import Q4Tensor
from usaf_amd.q4 import q4_linear

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]
IDS = dict(ids=lambda d: str(d).replace("torch.", ""))


@pytest.mark.parametrize("dtype", DTYPES, **IDS)
@pytest.mark.parametrize("m,n,k", [(1, 96, 640), (16, 64, 128), (96, 96, 640), (300, 257, 384), (1411, 1411, 256), (64, 192, 8192),
                                   (2049, 64, 128), (18, 1000, 1920), (70, 4100, 1024)])
def test_weights_are_the_codecs_bit_for_bit(m, n, k, dtype):
    """Rows with a single 1: a row of dx, a column of the output is one of the weight.  Scales over fp16's whole range, as far as
    15 of them stay finite: an infinite weight would make the others' zeros NaN."""
    q, s, z = O.codes(n, k, 9)
    s[5:60:2] = torch.logspace(-7, 3.6, 28).half()
    s[6:20:4] *= -1
    s[:2] = 0
    z[10:20] = 0
    z[20:24] = torch.tensor([-60000.0, 2.0 ** -24, -(2.0 ** -24), 1000.0]).half()
    w = Q4Tensor(q.cuda(), s.cuda(), z.cuda(), torch.Size((n, k)))
    values = O.weight(q, s, z, n, k, dtype).to(dtype).cuda()
    assert bool(torch.isfinite(values).all())
    for first in (0, max(n - m, 0)):
        at = (first + torch.arange(m)) % n
        dy = torch.zeros(m, n, dtype=dtype, device="cuda")
        dy[torch.arange(m), at] = 1
        x = torch.zeros(m, k, dtype=dtype, device="cuda", requires_grad=True)
        q4_linear(x, w).backward(dy)
        assert torch.equal(x.grad, values[at.cuda()])
    for first in (0, max(k - m, 0)):
        at = (first + torch.arange(m)) % k
        x = torch.zeros(m, k, dtype=dtype, device="cuda")
        x[torch.arange(m), at] = 1
        assert torch.equal(q4_linear(x, w), values[:, at.cuda()].t())


@pytest.mark.parametrize("dtype", DTYPES, **IDS)
@pytest.mark.parametrize("case", [c for c in P.CASES if c[0] == "gated16" and c[1] < 17000], ids=lambda c: "-".join(map(str, c[:5])))
def test_gated_of_whole_numbers(case, dtype):
    """Gates of 0 and 32, whose sigmoids are 1/2 and, in fp32, 1; ups of -3 to 3: what is kept, dG = d u s and dU = d g s are exact
    in 16 bits (and gate and up in the 8-bit blocks' 4), every sum in fp32."""
    _, m, inter, k, checkpoint, plans = case
    assert P.plans(*case[:5]) == plans
    gen = torch.Generator().manual_seed(m + k)
    left = k // 2  # columns with the gates' values; up reads the others
    x = torch.randint(-3, 4, (m, k), generator=gen).double()
    x[:, :left] = 32 * torch.randint(0, 2, (m, left), generator=gen)
    w = torch.zeros(2 * inter, k, dtype=torch.float64)
    w[torch.arange(inter), torch.randint(0, left, (inter,), generator=gen)] = 1
    w[inter + torch.arange(inter), torch.randint(left, k, (inter,), generator=gen)] = 1
    d = torch.randint(-2, 3, (m, inter), generator=gen).double() / 64
    x, w, d = (t.cuda() for t in (x, w, d))
    g, u = x @ w[:inter].t(), x @ w[inter:].t()
    s = torch.where(g == 0, 0.5, 1.0)
    dgu = torch.cat([d * u * s, d * g * s], 1)
    xg, wg = x.to(dtype).requires_grad_(), w.to(dtype).requires_grad_()
    y = gated_linear(xg, wg, checkpoint)
    y.backward(d.to(dtype))
    assert torch.equal(y.double(), g * s * u)
    # a sum is exact in fp32, in any order, while its magnitudes add up to less than 2^24 of the step that all its terms are
    # multiples of: 1/128 for dG (a half of d u), 1/2 for dU (32 d), 1 for x and for w, 32 for x's columns of gates
    steps = torch.full((2 * inter, 1), 2.0 ** -7, dtype=torch.float64, device="cuda")
    steps[inter:] = 0.5
    of_x = torch.ones(1, k, dtype=torch.float64, device="cuda")
    of_x[:, :left] = 32
    for got, a, b, step in ((xg.grad, dgu, w, 2.0 ** -7), (wg.grad, dgu.t(), x, steps * of_x)):
        assert float((a.abs() @ b.abs() / step).max()) < 2 ** 24
        assert torch.equal(got, (a @ b).to(dtype))
