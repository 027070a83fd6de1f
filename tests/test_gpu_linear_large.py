"""Weights of more than 4 GiB through the 4-bit product and the gated projection, forward and backward: rows at both ends and
around the places where 32-bit offsets would turn."""
import pytest
import torch

import linear_oracle as O
from fp8_oracle import half_step
from usaf_amd.gated import gated_linear
from usaf_amd.moe import Q4Tensor
from usaf_amd.q4 import q4_linear

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def room():
    if torch.cuda.mem_get_info()[0] < 120 << 30:
        pytest.skip("not enough memory")
    yield
    torch.cuda.empty_cache()


def _weight(rows, k):
    gen = torch.Generator("cuda").manual_seed(rows)
    n = rows * k // 128
    q = torch.randint(0, 256, (n, 64), dtype=torch.uint8, device="cuda", generator=gen).view(torch.int8)
    s = (0.003 + 0.002 * torch.rand(n, device="cuda", generator=gen)).half()
    return Q4Tensor(q, s, (-7.5 * s.float()).half(), torch.Size((rows, k)))


def _rows(w, at, dtype):
    """float64 values of a few rows."""
    rows, k = w.shape
    parts = (t.view(rows, k // 128, -1)[at].cpu() for t in (w.q, w.s, w.z))
    q, s, z = parts
    return O.weight(q.reshape(-1, 64), s.reshape(-1), z.reshape(-1), len(at), k, dtype)


def _around(rows, row_bytes):
    """The first and last rows and those at whole 2 GiB of the weight."""
    at = {0, 1, rows // 2, rows - 2, rows - 1}
    for gib in range(2, rows * row_bytes >> 30, 2):
        at |= {(gib << 30) // row_bytes + d for d in (-1, 0, 1)}
    return torch.tensor(sorted(a for a in at if a < rows), device="cuda")


def _x(m, k, dtype, seed=1):
    return torch.randn(m, k, device="cuda", generator=torch.Generator("cuda").manual_seed(seed)).to(dtype)


@pytest.mark.parametrize("m", [1, 20, 40, 600])
def test_product(m):
    n, k, dtype = 1_200_003, 8192, torch.bfloat16
    w = _weight(n, k)
    at = _around(n, k // 2)
    w64 = _rows(w, at, dtype)
    x = _x(m, k, dtype).requires_grad_()
    y = q4_linear(x, w)
    ref, off = O.product(x.detach().double().cpu(), w64)
    O.within(y[:, at], ref, O.rounded(ref, off, dtype), "out")
    dy = torch.zeros_like(y)
    dy[:, at] = _x(m, len(at), dtype, seed=2)
    y.backward(dy)
    ref, off = O.product(dy[:, at].double().cpu(), w64.t().contiguous())
    O.within(x.grad, ref, O.rounded(ref, off, dtype), "dx")


def _check_gated(y, x, weight, at, w64, dy, dtype):
    _, _, (act, off) = O.gated(x.detach().double().cpu(), w64)
    O.within(y[:, at], act, O.rounded(act, off, dtype), "act")
    y.backward(dy)
    (g, _), (u, _), _ = O.gated(x.detach().double().cpu(), w64)
    (dg, _), (du, _) = O.gated_grads(dy[:, at].double().cpu(), g, u)
    dgu = torch.cat([dg, du], 1)
    # dG and dU react to the roundings of what is kept by less than 3 times their share, and are rounded, and so is the result
    share = 5 * half_step(dtype)
    refs = [(x.grad, dgu @ w64)]
    if isinstance(weight, torch.Tensor):
        refs.append((weight.grad[torch.cat([at, at + y.shape[1]])], dgu.t() @ x.detach().double().cpu()))
    for got, ref in refs:
        assert float((got.double().cpu() - ref).norm()) <= share * float(ref.norm())


@pytest.mark.parametrize("m", [1, 40, 600])
def test_gated_4bit(m):
    """A gate of just below 4 GiB of codes: the up rows' offsets use all 32 bits."""
    inter, k, dtype = 1_048_000, 8192, torch.bfloat16
    assert 4 << 30 > (inter + 256) * (k // 2) > 15 << 28
    w = _weight(2 * inter, k)
    at = _around(inter, k // 2)
    w64 = _rows(w, torch.cat([at, at + inter]), dtype)
    x = _x(m, k, dtype).requires_grad_()
    with torch.no_grad():
        _, _, (act, off) = O.gated(x.double().cpu(), w64)
        O.within(gated_linear(x, w)[:, at], act, O.rounded(act, off, dtype), "act without a gradient")
    y = gated_linear(x, w)
    dy = torch.zeros_like(y)
    dy[:, at] = _x(m, len(at), dtype, seed=2)
    _check_gated(y, x, w, at, w64, dy, dtype)


@pytest.mark.parametrize("m,inter", [(64, 160_000), (37, 150_001), (1024, 160_000)])
def test_gated_16bit(m, inter):
    k, dtype = 8192, torch.bfloat16
    weight = (_x(2 * inter, k, dtype, seed=5) * 0.02).requires_grad_()
    at = _around(inter, 2 * k)
    w64 = weight.detach()[torch.cat([at, at + inter])].double().cpu()
    x = _x(m, k, dtype).requires_grad_()
    y = gated_linear(x, weight)
    dy = torch.zeros_like(y)
    dy[:, at] = _x(m, len(at), dtype, seed=2)
    _check_gated(y, x, weight, at, w64, dy, dtype)
    rest = torch.ones(2 * inter, dtype=torch.bool, device="cuda")
    rest[torch.cat([at, at + inter])] = False
    assert not weight.grad[rest].any()
