"""Gradients of the gated projection with a trained weight, at sizes whose products read operands with the contraction's index
first: columns that end inside a tile and a chunk of a line, contractions in parts, rows far apart."""
import pytest
import torch

import linear_oracle as O
import test_gpu_gated as T
from usaf_amd import _native as N
from usaf_amd import gated as G

pytestmark = pytest.mark.gpu
# tokens, intermediate, hidden: whole blocks of 64 tokens or not, of 2 I or not, hidden sizes in 8 or not
SIZES = [(64, 32, 8), (64, 32, 16), (128, 96, 200), (192, 160, 136), (320, 480, 1000), (128, 100, 264), (64, 2080, 72), (100, 96, 256),
         (1024, 64, 520), (448, 32, 1160), (640, 352, 248), (256, 33, 128), (576, 224, 132), (4160, 32, 24)]
# sizes at which dx's weight, dW's operands are read where they are
TURNED = [(1024, 64, 520, True, False), (512, 2080, 520, False, True), (448, 1600, 1160, False, True), (1088, 1056, 2056, True, True),
          (2112, 800, 1288, True, True), (640, 3520, 1288, True, True), (192, 8224, 1000, True, True)]


def _turned(m, inter, k):
    """From the workspaces: whether there is no room for copies of dx's weight, of dW's operands."""
    def up(v, to):
        return -(-v // to) * to
    lib, dgu = N.load(), up(2 * m * up(2 * inter, 64), 256)
    dx, dw = (lib.usaf_hip_gated_ws_bytes(m, inter, k, 0, what) - dgu for what in (1, 2))
    return dx < 2 * k * up(2 * inter, 64), dw < 2 * (2 * inter + k) * up(m, 64)


@pytest.mark.parametrize("dtype", T.DTYPES, ids=T._ids)
@pytest.mark.parametrize("m,inter,k", SIZES)
def test_gradients(m, inter, k, dtype):
    w = T._rand(2 * inter, k, dtype=dtype, seed=5, scale=0.1)
    x = T._rand(m, k, dtype=dtype).cuda().requires_grad_()
    T._check(G, x, w.cuda().requires_grad_(), w.double(), "fp8" if inter % 64 else None, dtype,
             T._rand(m, inter, dtype=dtype, seed=2))


@pytest.mark.parametrize("dtype", T.DTYPES, ids=T._ids)
@pytest.mark.parametrize("m,inter,k,dx,dw", TURNED)
def test_gradients_of_operands_where_they_are(m, inter, k, dx, dw, dtype):
    assert _turned(m, inter, k) == (dx, dw)
    test_gradients(m, inter, k, dtype)


@pytest.mark.parametrize("k,ld", [(264, 264), (264, 1024), (264, 301), (520, 4096)])
def test_rows_apart_and_single_gradients(k, ld):
    _rows_apart(256, 160, k, ld)


@pytest.mark.parametrize("ld", [1288, 4096, 1301])
def test_rows_apart_where_they_are(ld):
    assert _turned(2112, 800, 1288) == (True, True)
    _rows_apart(2112, 800, 1288, ld)


def _rows_apart(m, inter, k, ld):
    dtype = torch.bfloat16
    w = T._rand(2 * inter, k, dtype=dtype, seed=5, scale=0.1).cuda().requires_grad_()
    x = T._rand(m, k, dtype=dtype).cuda()
    dact = T._rand(m, inter, dtype=dtype, seed=2).cuda()
    xg = x.clone().requires_grad_()
    dx, dw = torch.autograd.grad(G.gated_linear(xg, w), (xg, w), dact)
    far = torch.full((m, ld), float("nan"), dtype=dtype, device="cuda")[:, :k]
    far.copy_(x)
    assert torch.equal(torch.autograd.grad(G.gated_linear(far, w), w, dact)[0], dw)  # the weight's alone
    assert torch.equal(torch.autograd.grad(G.gated_linear(xg, w.detach()), xg, dact)[0], dx)  # the rows' alone
    y = G.gated_linear(far.requires_grad_(), w)
    both = torch.autograd.grad(y, (far, w), dact)
    assert torch.equal(both[0], dx) and torch.equal(both[1], dw)


@pytest.mark.parametrize("m,inter,k", [(192, 96, 200), (640, 3520, 1288), (1088, 1056, 2056)])
def test_rows_that_are_not_finite_stay_alone(m, inter, k):
    dtype = torch.bfloat16
    w = T._rand(2 * inter, k, dtype=dtype, seed=5, scale=0.1).cuda()
    x = T._rand(m, k, dtype=dtype).cuda().requires_grad_()
    dact = T._rand(m, inter, dtype=dtype, seed=2).cuda()
    want = torch.autograd.grad(G.gated_linear(x, w), x, dact)[0]
    dact[70] = float("inf")
    dact[191, 3] = float("nan")
    got = torch.autograd.grad(G.gated_linear(x, w), x, dact)[0]
    rest = [i for i in range(m) if i not in (70, 191)]
    assert torch.equal(got[rest], want[rest])
    assert not torch.isfinite(got[70]).any() and torch.isnan(got[191]).all()


def test_whole_numbers_are_exact():
    """Products and sums that fp32 holds exactly: every place of both operands is where it belongs."""
    for m, inter, k in ((512, 320, 776), (64, 1056, 264), (1088, 32, 520), (1088, 1056, 2056), (640, 3520, 1288)):
        gen = torch.Generator().manual_seed(m)
        x = torch.randint(-3, 4, (m, k), generator=gen).bfloat16()
        w = torch.zeros(2 * inter, k, dtype=torch.bfloat16)
        w[torch.arange(2 * inter), torch.randint(0, k, (2 * inter,), generator=gen)] = 1
        dact = torch.randint(-2, 3, (m, inter), generator=gen).bfloat16()
        xg, wg = x.cuda().requires_grad_(), w.cuda().requires_grad_()
        dx, dw = torch.autograd.grad(G.gated_linear(xg, wg), (xg, wg), dact.cuda())
        x64, w64 = x.double(), w.double()
        g, u = x64 @ w64[:inter].t(), x64 @ w64[inter:].t()
        (dg, _), (du, _) = O.gated_grads(dact.double(), g, u)
        dgu = torch.cat([dg, du], 1)
        # dG and dU: bf16 of values with 2^-20 of their own error; the products' sums are far below their neighbours' steps
        slack = 2.0 ** -8 + 2.0 ** -18
        for got, ref, size in ((dx, dgu @ w64, dgu.abs() @ w64.abs()), (dw, dgu.t() @ x64, dgu.abs().t() @ x64.abs())):
            assert bool(((got.double().cpu() - ref).abs() <= 2 * slack * size + 1e-30).all())


@pytest.mark.parametrize("m,inter,k", [(128, 64, 64), (1088, 1056, 2056)])
def test_rows_off_16_bytes(m, inter, k):
    """The C entry: refused where x is read in place, taken where it is copied."""
    t = torch.zeros(m * k + 8, dtype=torch.bfloat16, device="cuda")
    dact = torch.zeros(m, inter, dtype=torch.bfloat16, device="cuda")
    kept = torch.zeros(m, 2, inter, dtype=torch.bfloat16, device="cuda")
    w = torch.zeros(2 * inter, k, dtype=torch.bfloat16, device="cuda")
    lib = N.load()
    need = lib.usaf_hip_gated_ws_bytes(m, inter, k, 0, 2)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")

    def call(x):
        return lib.usaf_hip_gated_bwd(dact.data_ptr(), N.dtype_code(t.dtype), m, inter, k, kept.data_ptr(), None, None, None,
                                      w.data_ptr(), x, k, None, w.data_ptr(), ws.data_ptr(), need, N.stream_ptr(t.device))

    assert call(t.data_ptr()) == 0
    assert call(t.data_ptr() + 2) == (1 if _turned(m, inter, k)[1] else 0)
    torch.cuda.synchronize()
