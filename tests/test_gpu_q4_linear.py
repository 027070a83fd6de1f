"""The product with a 4-bit weight on the GPU against the 64-bit oracle: values, grad-input, layouts, streams, graphs."""
import pytest
import torch

import linear_oracle as O
from fp8_oracle import half_step
from usaf_amd import _native as N

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]
# one row to many, every kind of tile's border; both sides of the sizes at which the weight is multiplied as codes
SIZES = [(1, 1, 128), (1, 64, 256), (2, 5, 128), (3, 4096, 2048), (7, 130, 384), (16, 48, 4096), (17, 33, 512), (31, 257, 640),
         (32, 96, 1024), (33, 128, 256), (64, 96, 384), (65, 1411, 256), (100, 520, 2944), (129, 255, 1024), (300, 384, 512),
         (257, 640, 1920), (511, 96, 256), (512, 130, 128), (513, 300, 896), (1030, 530, 384), (2049, 64, 128),
         (8, 33, 4096), (16, 300, 2048), (1, 40, 14336), (5, 1000, 1920), (1, 9000, 256), (100, 64, 14336), (700, 192, 8192)]


def _ids(d):
    return str(d).replace("torch.", "")


@pytest.fixture(scope="module")
def L():
    from usaf_amd import q4
    return q4


def _weight(rows, k, seed=0):
    from usaf_amd.moe import Q4Tensor
    parts = O.codes(rows, k, seed)
    return Q4Tensor(*(t.cuda() for t in parts), torch.Size((rows, k))), parts


def _x(m, k, dtype, seed=1):
    return torch.randn(m, k, generator=torch.Generator().manual_seed(seed)).to(dtype)


@pytest.mark.parametrize("dtype", DTYPES, ids=_ids)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_product_and_gradient(L, m, n, k, dtype):
    w, parts = _weight(n, k, seed=m + n)
    w64 = O.weight(*parts, n, k, dtype)
    x, dy = _x(m, k, dtype), _x(m, n, dtype, seed=2)
    xg = x.cuda().requires_grad_()
    y = L.q4_linear(xg, w)
    assert y.dtype == dtype
    ref, off = O.product(x.double(), w64)
    O.within(y, ref, O.rounded(ref, off, dtype), "out")
    y.backward(dy.cuda())
    ref, off = O.product(dy.double(), w64.t().contiguous())
    O.within(xg.grad, ref, O.rounded(ref, off, dtype), "dx")
    with torch.no_grad():
        assert torch.equal(L.q4_linear(x.cuda(), w), y)


@pytest.mark.parametrize("dtype", DTYPES, ids=_ids)
@pytest.mark.parametrize("m", [1, 5, 32, 128, 640])
def test_weights_are_the_codecs_bit_for_bit(L, m, dtype):
    """Rows with a single 1: an output is one weight.  Scales up to where code * scale overflows fp16, and tiny ones."""
    n, k = 96, 640
    w, (q, s, z) = _weight(n, k, seed=9)
    w.s[5:40] = torch.logspace(-7, 4, 35).half().cuda()
    w.z[10:20] = 0
    values = w.dequantize(dtype)
    fine = torch.isfinite(values).all(1)
    for first in range(0, k, m):
        x = torch.zeros(m, k, dtype=dtype)
        rows = range(min(m, k - first))
        for r in rows:
            x[r, first + r] = 1
        y = L.q4_linear(x.cuda(), w)
        assert torch.equal(y[:len(rows)][:, fine], values.t()[first:first + len(rows)][:, fine])
        dx = torch.zeros(m, k, dtype=dtype).cuda().requires_grad_()
        dy = torch.zeros(m, n, dtype=dtype)
        for r in range(min(m, n)):
            dy[r, r] = 1
        L.q4_linear(dx, w).backward(dy.cuda())
        keep = fine.nonzero().view(-1)
        keep = keep[keep < m]
        if bool(fine.all()):
            assert torch.equal(dx.grad[keep], values[keep])
        if m >= 128:
            break


def test_differences(L):
    """The product is linear: (f(x + v) - f(x)) . dy = v . dx up to the outputs' roundings, for x and v on a grid that fp16
    holds exactly."""
    m, n, k = 40, 130, 256
    w, parts = _weight(n, k)
    gen = torch.Generator().manual_seed(4)
    x, v = (torch.randint(-8, 9, (m, k), generator=gen).double() / 8 for _ in range(2))
    dy = torch.randint(-8, 9, (m, n), generator=gen).double() / 8
    xg = x.half().cuda().requires_grad_()
    y0 = L.q4_linear(xg, w)
    y0.backward(dy.half().cuda())
    y1 = L.q4_linear((x + v).half().cuda(), w)
    lhs = ((y1.double().cpu() - y0.detach().double().cpu()) * dy).sum()
    rhs = (v * xg.grad.double().cpu()).sum()
    w64 = O.weight(*parts, n, k, torch.float16)
    room = sum((O.rounded(*O.product(a, w64), torch.float16) * dy.abs()).sum() for a in (x, x + v))
    ref, off = O.product(dy, w64.t().contiguous())
    room = room + (O.rounded(ref, off, torch.float16) * v.abs()).sum()
    assert abs(float(lhs - rhs)) <= float(room)


@pytest.mark.parametrize("dtype", DTYPES, ids=_ids)
@pytest.mark.parametrize("m,n,k", [(4, 1024, 2048), (200, 512, 1024), (1024, 512, 1024)])
def test_nothing_but_the_last_rounding_shows(L, m, n, k, dtype):
    """On normal data the distance to the exact product is that of the rounding alone (half a step, rms a third of its
    square), with a tenth on top."""
    w, parts = _weight(n, k)
    w64 = O.weight(*parts, n, k, dtype)
    x = _x(m, k, dtype)
    ref = x.double() @ w64.t()
    alone = O.rms_off(ref.to(dtype), ref)
    assert O.rms_off(L.q4_linear(x.cuda(), w), ref) <= 1.1 * alone <= 1.1 * half_step(dtype)


def test_shapes_strides_and_empty_calls(L):
    w, _ = _weight(130, 256)
    x = _x(24, 256, torch.bfloat16).cuda()
    y = L.q4_linear(x, w)
    assert torch.equal(L.q4_linear(x.view(2, 3, 4, 256), w), y.view(2, 3, 4, 130))
    assert torch.equal(L.q4_linear(x[0], w), L.q4_linear(x[:1], w)[0])
    wide = torch.zeros(24, 300, dtype=torch.bfloat16, device="cuda")
    for first in (0, 8, 3):  # rows 16-byte aligned, and not
        wide[:, first:first + 256] = x
        assert torch.equal(L.q4_linear(wide[:, first:first + 256], w), y)
    odd = torch.zeros(24, 257, dtype=torch.bfloat16, device="cuda")
    odd[:, 1:] = x
    assert torch.equal(L.q4_linear(odd[:, 1:], w), y)
    assert torch.equal(L.q4_linear(x.t().contiguous().t(), w), y)
    assert torch.equal(L.q4_linear(x[:1].expand(24, 256), w), y[:1].expand(24, 130))
    assert torch.equal(L.q4_linear(x[::2], w), y[::2]) and torch.equal(L.q4_linear(x.flip(0), w), y.flip(0))
    for shape in [(0, 256), (2, 0, 256)]:
        e = torch.zeros(*shape, dtype=torch.float16, device="cuda", requires_grad=True)
        out = L.q4_linear(e, w)
        assert out.shape == (*shape[:-1], 130)
        out.sum().backward()
        assert e.grad.shape == e.shape
    # gradients that are expanded, transposed, of another type's sum
    xg = x.clone().requires_grad_()
    L.q4_linear(xg, w).sum().backward()
    first = xg.grad.clone()
    xg.grad = None
    L.q4_linear(xg, w).backward(torch.ones(130, 24, dtype=torch.bfloat16, device="cuda").t())
    assert torch.equal(first, xg.grad)


@pytest.mark.parametrize("m", [1, 9, 40, 200, 600])
def test_rows_that_are_not_finite_stay_alone(L, m):
    w, _ = _weight(257, 512)
    x = _x(m, 512, torch.float16)
    y = L.q4_linear(x.cuda(), w)
    bad = x.clone()
    bad[m // 2, 7] = float("nan")
    z = L.q4_linear(bad.cuda(), w)
    assert bool(torch.isnan(z[m // 2]).all())
    keep = torch.arange(m) != m // 2
    assert torch.equal(z[keep.cuda()], y[keep.cuda()])


def test_two_streams_and_repeats(L):
    w, _ = _weight(1411, 512)
    xs = [_x(m, 512, torch.bfloat16, seed=m).cuda() for m in (1, 37, 300, 700)]
    ref = [L.q4_linear(x, w) for x in xs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for rep in range(4):
        for i, x in enumerate(xs):
            with torch.cuda.stream(streams[(i + rep) % 2]):
                outs.append((i, L.q4_linear(x, w)))
    torch.cuda.synchronize()
    assert all(torch.equal(ref[i], y) for i, y in outs)


def test_in_a_graph(L):
    w, _ = _weight(640, 1024)
    cold, _ = _weight(640, 1024)
    for m in (1, 40, 600):
        x = _x(m, 1024, torch.bfloat16).cuda()
        with torch.no_grad():
            L.q4_linear(x, w)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                y = L.q4_linear(L.q4_linear(x, w)[:, :512].repeat(1, 2), w)
            for seed in range(3):
                x.copy_(_x(m, 1024, torch.bfloat16, seed=seed + 10))
                want = L.q4_linear(L.q4_linear(x, w)[:, :512].repeat(1, 2), w)
                graph.replay()
                torch.cuda.synchronize()
                assert torch.equal(y, want)
    x = _x(4, 1024, torch.bfloat16).cuda()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        z = x * 2
        with pytest.raises(RuntimeError, match="captured"):
            L.q4_linear(x, cold)
        with pytest.raises(RuntimeError, match="captured"):
            L.q4_linear(x.requires_grad_(), w)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(z, x.detach() * 2)


def test_second_derivatives_tangents_and_traces(L):
    w, _ = _weight(64, 128)
    x = _x(3, 128, torch.float16).cuda().requires_grad_()
    with pytest.raises(RuntimeError, match="second"):
        torch.autograd.grad(L.q4_linear(x, w).sum(), x, create_graph=True)
    from torch.autograd import forward_ad
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x.detach(), torch.ones_like(x))
        with pytest.raises((RuntimeError, NotImplementedError)):
            L.q4_linear(dual, w)
    plain = x.detach()
    traced = torch.jit.trace(lambda t: L.q4_linear(t, w), (plain,), check_trace=False)
    assert torch.equal(traced(plain * 2), L.q4_linear(plain * 2, w))


def test_workspaces_that_are_too_small(L):
    w, _ = _weight(256, 256)
    x, sz = _x(600, 256, torch.float16).cuda(), L.words("", w)
    out = torch.empty(600, 256, dtype=torch.float16, device="cuda")
    need = N.load().usaf_hip_q4_linear_ws_bytes(600, 256, 256, 1)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    for size in (0, need - 1):
        with pytest.raises(ValueError, match="workspace"):
            N.call("usaf_hip_q4_linear_bwd", x.data_ptr(), N.F16, 600, 256, 256, w.q.data_ptr(), sz.data_ptr(), 256,
                   out.data_ptr(), ws.data_ptr(), size, N.stream_ptr(x.device))
