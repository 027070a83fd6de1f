"""Which of the 8-bit products sum to fp32's precision: gate and up, the gated activation's gradient, a few rows.

The 8-bit matrix instruction drops what lies far below the largest of its 64 products; the 16-bit one keeps it.  The
products whose results are quantized again, and those of a few rows, take the second."""
import pytest
import torch

import fp8_oracle as O
from usaf_amd import _native as N

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]


def _ids(d):
    return str(d).replace("torch.", "")


@pytest.fixture(scope="module")
def F():
    from usaf_amd import fp8
    return fp8


def _rand(*shape, dtype=torch.bfloat16, seed=0, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def _within(got, ref, bound):
    off = (got.detach().double().cpu() - ref).abs() - bound
    assert got.shape == ref.shape and float(off.max()) <= 0, f"{float(off.max())} past the bound"


def _product(F, x, w, out, offsets=None):
    E, n, k = (1, *w.shape) if len(w.shape) == 2 else w.shape
    r = F.quantize_rows(x)
    N.call("usaf_hip_fp8_gemm", r.q.data_ptr(), r.s.data_ptr(), x.shape[0], None, out.shape[0], w.q.data_ptr(), w.s.data_ptr(),
           N.ptr(offsets), E, n, k, N.dtype_code(out.dtype), 1, out.data_ptr(), N.stream_ptr(out.device))


# 32 x 32 to 256 x 256 tiles, and the contraction split over a block's waves
SIZES = [(5, 40, 300), (70, 500, 640), (300, 1411, 520), (500, 4100, 256), (2000, 4100, 256)]


@pytest.mark.parametrize("dtype", DTYPES, ids=_ids)
@pytest.mark.parametrize("M,N_,K", SIZES)
def test_wide_product(F, M, N_, K, dtype):
    x, w = _rand(M, K, dtype=dtype, seed=M), _rand(N_, K, dtype=torch.float32, seed=N_, scale=0.05)
    out = torch.empty(M, N_, dtype=dtype, device="cuda")
    _product(F, x.cuda(), F.Fp8Tensor.quantize(w.cuda()), out)
    a, wq = O.quantized_rows(x)[0], O.quantized_weight(w)[0]
    ref = a @ wq.t()
    _within(out, ref, O.wide_bound(a, wq, ref, dtype))


# rows * ceil(K / 128) * 128 <= 16,384, at most 32 rows: one launch, which quantizes the rows itself
@pytest.mark.parametrize("dtype", DTYPES, ids=_ids)
@pytest.mark.parametrize("M,N_,K", [(1, 4096, 2048), (1, 70, 16001), (8, 4100, 2000), (17, 33, 300), (32, 8200, 512), (5, 9001, 384)])
def test_linear_of_a_few_rows(F, M, N_, K, dtype):
    x, w = _rand(M, K, dtype=dtype, seed=M), _rand(N_, K, dtype=torch.float32, seed=N_, scale=0.05)
    out = F.fp8_linear(x.cuda(), F.Fp8Tensor.quantize(w.cuda()))
    a, wq = O.quantized_rows(x)[0], O.quantized_weight(w)[0]
    ref = a @ wq.t()
    _within(out, ref, O.wide_bound(a, wq, ref, dtype))


def _cancelling(rows, cols, K):
    """x [rows, K], w [cols, K] whose product is whole numbers: in every 64 of the contraction a pair of 2^16 that cancels and
    62 products of 2, each 2^-15 of it.  All are codes with a scale of 1, and the sum is exact in fp32."""
    x, w = torch.ones(rows, K), torch.full((cols, K), 2.0)
    x[:, 3::64], x[:, 40::64] = 256, -256
    w[:, 3::64], w[:, 40::64] = 256, 256
    x[1::2] *= -1
    return x, w, x.double() @ w.double().t()


def _rounded(ref, dtype):
    return ref.to(dtype).double()


@pytest.mark.parametrize("dtype", DTYPES, ids=_ids)
@pytest.mark.parametrize("M,N_,K", SIZES[:-1])
def test_wide_product_keeps_what_is_small_beside_a_pair_that_cancels(F, M, N_, K, dtype):
    K = K // 64 * 64
    x, w, ref = _cancelling(M, N_, K)
    out = torch.empty(M, N_, dtype=dtype, device="cuda")
    _product(F, x.to(dtype).cuda(), F.Fp8Tensor.quantize(w.cuda()), out)
    assert torch.equal(out.double().cpu(), _rounded(ref, dtype)) and float(ref.abs().min()) == 124 * (K // 64)


@pytest.mark.parametrize("dtype", DTYPES, ids=_ids)
@pytest.mark.parametrize("M", [1, 8, 32])
def test_a_few_rows_keep_it(F, M, dtype):
    x, w, ref = _cancelling(M, 300, 512)
    out = F.fp8_linear(x.to(dtype).cuda(), F.Fp8Tensor.quantize(w.cuda()))
    assert torch.equal(out.double().cpu(), _rounded(ref, dtype))


@pytest.mark.parametrize("dtype", DTYPES, ids=_ids)
@pytest.mark.parametrize("T,E,H,I", [(40, 2, 256, 128), (700, 2, 128, 256)])
def test_the_experts_inner_products_keep_it(F, T, E, H, I, dtype):
    """Gate and up, and d(act): through the layer's own calls."""
    from usaf_amd import moe as G
    hs, wgu, ref = _cancelling(T, 2 * I, H)
    dout, wd_t, dref = _cancelling(T, I, H)  # d(act)[t, i] = sum_h dout[t, h] wd[h, i], every routing weight 1
    wgu, wd = wgu.expand(E, 2 * I, H).contiguous(), wd_t.t().expand(E, H, I).contiguous()
    ew = G.ExpertWeights(F.Fp8Tensor.quantize(wgu.cuda()), F.Fp8Tensor.quantize(wd.cuda()))
    weights = torch.zeros(T, E, dtype=dtype, device="cuda")
    weights[torch.arange(T), torch.arange(T) % E] = 1
    hv = hs.to(dtype).cuda().requires_grad_(True)
    out = G.routed_experts(hv, weights, ew)
    _, gu, _, y = out.grad_fn.saved_tensors
    b = out.grad_fn.b
    tok = b.token_idx.long().cpu()
    assert torch.equal(gu.double().cpu(), _rounded(ref, dtype)[tok])
    # a gate of 32 has silu(32) = 32 and a slope of 1 in fp32 (exp(-32) is 2^-46), up of 1: dgu = (d(act), 32 d(act))
    given = torch.cat([torch.full((T, I), 32.0), torch.ones(T, I)], 1).to(dtype).cuda()
    dgu = torch.empty_like(given)
    F.experts_bwd(dout.to(dtype).cuda(), y, given, ew, b, None, dgu, torch.zeros(T, E, dtype=dtype, device="cuda"))
    dact = _rounded(dref, dtype)[tok]
    assert torch.equal(dgu.double().cpu(), torch.cat([dact, 32 * dact], 1))


@pytest.mark.parametrize("dtype", DTYPES, ids=_ids)
def test_the_experts_gate_and_up(F, dtype):
    """On normal data, without the 8-bit instruction's allowance."""
    from usaf_amd import moe as G
    T, E, H, I = 200, 3, 256, 128
    wgu = _rand(E, 2 * I, H, dtype=torch.float32, seed=1, scale=0.05)
    ew = G.ExpertWeights(F.Fp8Tensor.quantize(wgu.cuda()), F.Fp8Tensor.quantize(_rand(E, H, I, seed=2, scale=0.05).cuda()))
    hs = _rand(T, H, dtype=dtype, seed=3)
    weights = torch.full((T, E), 0.25, dtype=dtype)
    out = G.routed_experts(hs.cuda().requires_grad_(True), weights.cuda(), ew)
    gu, offs, tok = out.grad_fn.saved_tensors[1], out.grad_fn.b.offsets.tolist(), out.grad_fn.b.token_idx.long().cpu()
    a, wq = O.quantized_rows(hs)[0], O.quantized_weight(wgu)[0]
    for e in range(E):
        s = slice(offs[e], offs[e + 1])
        ref = a[tok[s]] @ wq[e].t()
        _within(gu[s], ref, O.wide_bound(a[tok[s]], wq[e], ref, dtype))
