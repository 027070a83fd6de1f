"""8-bit block format on the GPU against the 64-bit oracle: codec, product, grad-input, routed experts."""
import pytest
import torch

import fp8_oracle as O
from usaf_amd import _native as N

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]


def _product(x, w, out, offsets=None, row_of=None, wide=False):
    """out[m] = x[row_of[m] or m] @ w_e^T for the slots m of expert e, as the layer's calls make it."""
    E, n, k = (1, *w.shape) if len(w.shape) == 2 else w.shape
    N.call("usaf_hip_fp8_gemm", x.q.data_ptr(), x.s.data_ptr(), x.q.shape[0], N.ptr(row_of), out.shape[0], w.q.data_ptr(),
           w.s.data_ptr(), N.ptr(offsets), E, n, k, N.dtype_code(out.dtype), 1 if wide else 0, out.data_ptr(),
           N.stream_ptr(out.device))


def _ids(d):
    return str(d).replace("torch.", "")


@pytest.fixture(scope="module")
def F():
    from usaf_amd import fp8
    return fp8


def _rand(*shape, dtype=torch.bfloat16, seed=0, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def _within(got, ref, bound):
    got = got.detach().double().cpu()
    assert got.shape == ref.shape
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    fine = torch.isfinite(ref)
    off = ((got - ref).abs() - bound)[fine]
    assert off.numel() == 0 or float(off.max()) <= 0, f"{float(off.max())} past the bound"


# ---- codec ---------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES, ids=_ids)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 127), (5, 128), (2, 129), (17, 640), (4, 2027), (9, 512), (5, 1536),
                                       (33, 2048)])
def test_quantize_rows_is_the_oracles(F, rows, cols, dtype):
    # magnitudes over the type's whole range, a row of zeros, a block border of every kind
    x = _rand(rows, cols, dtype=torch.float32, seed=rows + cols)
    x = (x * torch.exp2(torch.randint(-20, 12, (rows, cols), generator=torch.Generator().manual_seed(1)).float())).to(dtype)
    x[rows // 2] = 0
    r = F.quantize_rows(x.cuda())
    ref, e = O.quantized_rows(x)
    nb = -(-cols // 128)
    assert r.q.shape == (rows, nb * 128)
    s = r.s[:, :nb].cpu()
    live = ref.new_tensor(0) != torch.nn.functional.pad(ref, (0, -cols % 128)).view(rows, nb, 128).abs().amax(-1)
    assert torch.equal(s[live].int(), e[live].int())
    got = r.q.cpu().view(torch.float8_e4m3fn).double().view(rows, nb, 128) * torch.exp2(s.double() - 127)[..., None]
    got = got.view(rows, -1)
    assert torch.equal(got[:, :cols], ref) and not got[:, cols:].any()


@pytest.mark.parametrize("amax", [448.0, 449.0, 447.0, 896.0, 900.0, 1.75, 1.7578125, 2.0 ** -100, 3.0e38])
def test_scale_at_the_borders(F, amax):
    x = torch.zeros(1, 128, dtype=torch.bfloat16)
    x[0, 3], x[0, 77] = amax, -amax / 3
    r = F.quantize_rows(x.cuda())
    ref, e = O.quantized_rows(x)
    assert int(r.s[0, 0]) == int(e[0, 0])
    assert torch.equal(O.values(r.q.cpu(), r.s[:, :1].cpu(), (1, 128)), ref)
    assert float(x.abs().max()) * 2.0 ** (127 - int(r.s[0, 0])) <= 448


@pytest.mark.parametrize("cols", [256, 512, 2048])
def test_rows_behind_the_given_count_are_left(F, cols):
    x = _rand(23, cols).cuda()
    n = torch.tensor([4], dtype=torch.int32, device="cuda")
    rows = F.empty_rows(23, cols, x.device)
    rows.q.fill_(17)
    N.call("usaf_hip_fp8_quantize_rows", x.data_ptr(), N.BF16, 23, cols, cols, n.data_ptr(), rows.q.data_ptr(),
           rows.s.data_ptr(), N.stream_ptr(x.device))
    assert bool((rows.q[4:] == 17).all()) and torch.equal(rows.q[:4], F.quantize_rows(x[:4]).q)


@pytest.mark.parametrize("shape", [(1, 1), (128, 128), (130, 257), (3, 96, 200), (2, 256, 128)])
@pytest.mark.parametrize("dtype", [torch.float32] + DTYPES, ids=_ids)
def test_weight_codec_and_transpose(F, shape, dtype):
    w = _rand(*shape, dtype=dtype, seed=len(shape), scale=0.02)
    t = F.Fp8Tensor.quantize(w.cuda())
    ref, e = O.quantized_weight(w)
    assert torch.equal(t.s.cpu().int(), e.int())
    assert torch.equal(O.values(t.q.cpu(), t.s.cpu(), shape), ref)
    assert torch.equal(t.dequantize().cpu().double(), ref)
    assert torch.equal(t.dequantize(torch.bfloat16).cpu().double(), ref)
    tt = t.transposed()
    assert tt.shape == (*shape[:-2], shape[-1], shape[-2]) and tt is t.transposed()
    assert torch.equal(O.values(tt.q.cpu(), tt.s.cpu(), tt.shape), ref.transpose(-1, -2))
    assert not tt.q[..., shape[-2]:].any() and not t.q[..., shape[-1]:].any()


def test_values_that_are_not_finite(F):
    x = _rand(4, 300)
    x[1, 5], x[2, 200], x[3, 299] = float("inf"), float("nan"), float("-inf")
    w = F.Fp8Tensor.quantize(_rand(65, 300, seed=3, scale=0.1).cuda())
    y = F.fp8_linear(x.cuda(), w)
    assert bool(torch.isnan(y[1:]).all())
    assert torch.equal(y[:1], F.fp8_linear(x[:1].cuda(), w)) and bool(torch.isfinite(y[0]).all())
    v = _rand(130, 140)
    v[129, 139] = float("inf")
    t = F.Fp8Tensor.quantize(v.cuda())
    assert int(torch.isnan(t.dequantize()).sum()) == 1


# ---- product -------------------------------------------------------------------

SIZES = [(1, 1, 1), (1, 64, 128), (2, 5, 127), (7, 130, 129), (31, 257, 640), (33, 128, 256), (64, 96, 384), (65, 1411, 300),
         (129, 255, 1024), (300, 384, 512), (257, 640, 2027), (513, 300, 896)]
# ... and of the product for a few rows: one to 32 rows, one to four rounds of column tiles, short and long contractions
SIZES += [(8, 4100, 2000), (1, 70, 16001), (17, 33, 300), (32, 8200, 512), (5, 9001, 384), (1, 25000, 130), (16, 640, 1024)]


@pytest.mark.parametrize("dtype", DTYPES, ids=_ids)
@pytest.mark.parametrize("M,N,K", SIZES)
def test_linear(F, M, N, K, dtype):
    x, w = _rand(M, K, dtype=dtype, seed=M), _rand(N, K, dtype=torch.float32, seed=N, scale=0.05)
    t = F.Fp8Tensor.quantize(w.cuda())
    xv = x.cuda().requires_grad_(True)
    y = F.fp8_linear(xv, t)
    assert y.dtype == dtype
    a, wq = O.quantized_rows(x)[0], O.quantized_weight(w)[0]
    ref = a @ wq.t()
    _within(y, ref, O.product_bound(a, wq, ref, dtype))
    dy = _rand(M, N, dtype=dtype, seed=K)
    y.backward(dy.cuda())
    b = O.quantized_rows(dy)[0]
    ref = b @ wq
    _within(xv.grad, ref, O.product_bound(b, wq.t(), ref, dtype))
    assert torch.equal(F.fp8_linear(x.cuda(), t), y.detach())  # the same bits again, without a graph


@pytest.mark.parametrize("dtype", DTYPES, ids=_ids)
def test_linear_sums_whole_numbers_exactly(F, dtype):
    """Codes and scales that make every product and sum a whole number: no rounding anywhere, so a code at a wrong
    place cannot hide in a tolerance."""
    g = torch.Generator().manual_seed(5)
    x = torch.randint(-2, 3, (70, 512), generator=g).to(dtype)
    w = torch.randint(-1, 2, (200, 512), generator=g).float()
    ref = x.double() @ w.double().t()
    assert float(ref.abs().max()) <= 256  # whole numbers that bf16 holds
    assert torch.equal(F.fp8_linear(x.cuda(), F.Fp8Tensor.quantize(w.cuda())).double().cpu(), ref)


def test_scales_of_every_block_reach_the_product(F):
    """Blocks that differ by powers of two in every place of the exponent's range a sum in fp32 can hold."""
    x = torch.zeros(40, 1024, dtype=torch.bfloat16)
    w = torch.zeros(300, 1024)
    for kb in range(8):
        x[:, kb * 128 + 3 * kb] = 2.0 ** (kb - 4)
        w[:, kb * 128 + 3 * kb] = 2.0 ** (-2 * kb)
    x[::2] *= 4
    w[128:256] *= 0.5
    ref = x.double() @ w.double().t()
    assert torch.equal(F.fp8_linear(x.cuda(), F.Fp8Tensor.quantize(w.cuda())).double().cpu(), ref.bfloat16().double())


def test_gradient_against_differences(F):
    """The product is linear in x wherever x and x + h are codes: differences are exact there."""
    g = torch.Generator().manual_seed(7)
    M, N, K = 3, 140, 130
    x = torch.randint(-4, 5, (M, K), generator=g).to(torch.bfloat16)
    w = torch.randint(-2, 3, (N, K), generator=g).float()
    dy = torch.randint(-3, 4, (M, N), generator=g).to(torch.bfloat16)
    t = F.Fp8Tensor.quantize(w.cuda())
    xv = x.cuda().requires_grad_(True)
    F.fp8_linear(xv, t).backward(dy.cuda())
    for m, k in [(0, 0), (1, 64), (2, 127), (0, 128), (2, 129)]:
        up, down = x.clone(), x.clone()
        up[m, k] += 1
        down[m, k] -= 1
        d = (F.fp8_linear(up.cuda(), t).double() - F.fp8_linear(down.cuda(), t).double()) / 2
        assert float((d.cpu() * dy.double()).sum()) == float(xv.grad[m, k])


def test_linear_strides_shapes_and_streams(F):
    t = F.Fp8Tensor.quantize(_rand(72, 136, seed=2, scale=0.1).cuda())
    base = _rand(6, 5, 280, seed=4).cuda()
    for x in (base[:, :, 3:139], base[:, ::2, :136], base[:, :, :272:2], base[0, :1, :136].expand(4, 136),
              base[:3, 0, 1:137], base.permute(1, 0, 2)[:, :, 8:144], base[0, 0, :136]):
        want = F.fp8_linear(x.contiguous(), t)
        assert torch.equal(F.fp8_linear(x, t), want) and want.shape == (*x.shape[:-1], 72)
    assert F.fp8_linear(base[:0, 0, :136], t).shape == (0, 72)
    z = base[:0, 0, :136].clone().requires_grad_(True)
    F.fp8_linear(z, t).sum().backward()
    assert z.grad.shape == (0, 136)
    want = F.fp8_linear(base[:, :, :136], t)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = F.fp8_linear(base[:, :, :136], t)
    s.synchronize()
    assert torch.equal(got, want)


def test_linear_has_no_second_derivative(F):
    t = F.Fp8Tensor.quantize(_rand(64, 128).cuda())
    x = _rand(2, 128).cuda().requires_grad_(True)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(F.fp8_linear(x, t).sum(), x, create_graph=True)
    (g,) = torch.autograd.grad(F.fp8_linear(x, t).sum(), x)
    assert g.shape == x.shape


@pytest.mark.parametrize("rows", [3, 50])
def test_linear_in_a_graph(F, rows):
    t = F.Fp8Tensor.quantize(_rand(200, 384, seed=2, scale=0.1).cuda())
    x = _rand(rows, 384, seed=1).cuda()
    with torch.no_grad():
        F.fp8_linear(x, t)
        graphs = []
        for _ in range(2):  # two graphs of the same call: neither has the other's buffers
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                out = F.fp8_linear(x, t)
            graphs.append((g, out))
        for i in range(4):
            x.copy_(_rand(rows, 384, seed=10 + i))
            for g, out in graphs:
                g.replay()
                torch.cuda.synchronize()
                want = F.fp8_linear(x, t)
                torch.cuda.synchronize()
                assert torch.equal(out, want)


# ---- routed experts --------------------------------------------------------------

def _experts(F, E, H, I, seed=0):
    from usaf_amd.moe import ExpertWeights
    gu, dn = _rand(E, 2 * I, H, seed=seed, scale=0.05), _rand(E, H, I, seed=seed + 1, scale=0.05)
    return ExpertWeights(F.Fp8Tensor.quantize(gu.cuda()), F.Fp8Tensor.quantize(dn.cuda()))


def _routing(T, E, k, dtype, seed=0, only=None):
    g = torch.Generator().manual_seed(seed)
    p = torch.softmax(torch.randn(T, E, generator=g), -1)
    if only is not None:
        p[:, [e for e in range(E) if e not in only]] = 0
    top = p.topk(k, -1)
    return torch.zeros_like(p).scatter_(1, top.indices, top.values / top.values.sum(-1, keepdim=True)).to(dtype)


# few and many slots for an expert, experts without one, an uneven routing, one token
@pytest.mark.parametrize("dtype", DTYPES, ids=_ids)
@pytest.mark.parametrize("T,E,k,H,I,only", [(1, 4, 2, 128, 128, None), (40, 5, 2, 256, 384, None), (70, 3, 1, 384, 128, [1]),
                                            (300, 4, 2, 256, 256, None), (33, 200, 3, 128, 128, None),
                                            (700, 2, 2, 128, 256, None)])
def test_experts_step_by_step(F, T, E, k, H, I, only, dtype):
    """Every step of the forward and backward against 64 bits of what that step was given: a code that falls
    to the other side of a border in one step is the next one's input, not its error."""
    from usaf_amd import moe as G
    ew = _experts(F, E, H, I)
    hs, w = _rand(T, H, dtype=dtype, seed=9), _routing(T, E, k, dtype, seed=3, only=only)
    dout = _rand(T, H, dtype=dtype, seed=11)
    hv, wv = hs.cuda().requires_grad_(True), w.cuda().requires_grad_(True)
    out = G.routed_experts(hv, wv, ew)
    saved = out.grad_fn
    _, gu, act, y = saved.saved_tensors
    b = saved.b
    assert act is None  # no weight gradient is wanted
    act, again = torch.empty(b.n_slots, I, dtype=dtype, device="cuda"), torch.empty_like(gu)
    assert torch.equal(F.experts_forward(F.quantize_rows(hs.cuda()), ew, b, again, act, dtype), y) and torch.equal(again, gu)
    offs, tok = b.offsets.tolist(), b.token_idx.long().cpu()
    wgu, wd = ew.gate_up.dequantize().double().cpu(), ew.down.dequantize().double().cpu()
    h = O.half_step(dtype)
    a, q_act = O.quantized_rows(hs)[0], O.quantized_rows(act.cpu())[0]
    g64, u64 = gu.double().cpu().split(I, 1)
    sig = torch.sigmoid(g64)
    silu = g64 * sig
    # silu and its product are rounded one behind the other; silu_fast's exp2 and reciprocal are good to about 2^-22
    _within(act, silu * u64, (silu * u64).abs() * (2.01 * h + 2.0 ** -20) + O.tiny(dtype) * (1 + u64.abs()))
    for e in range(E):
        s = slice(offs[e], offs[e + 1])
        if offs[e] == offs[e + 1]:
            continue
        ref = a[tok[s]] @ wgu[e].t()
        _within(gu[s], ref, O.product_bound(a[tok[s]], wgu[e], ref, dtype))
        ref = q_act[s] @ wd[e].t()
        _within(y[s], ref, O.product_bound(q_act[s], wd[e], ref, dtype))
    y64, gu = y.double().cpu(), gu.clone()
    ref, mags = torch.zeros(T, H, dtype=torch.float64), torch.zeros(T, H, dtype=torch.float64)
    slot_e = torch.repeat_interleave(torch.arange(E), torch.tensor(offs[1:]) - torch.tensor(offs[:-1]))
    pw = w[tok, slot_e].double()[:, None]
    ref.index_add_(0, tok, pw * y64)
    mags.index_add_(0, tok, (pw * y64).abs())
    _within(out, ref, ref.abs() * h + O.tiny(dtype) + (E + 1) * 2.0 ** -24 * mags)
    out.backward(dout.cuda())
    # the backward's own steps again, on its inputs
    dcur64 = pw * dout[tok].double()
    dcur = dcur64.to(dtype).cuda()
    dgu, got_dcur, dweights = torch.empty_like(gu), torch.empty_like(y), torch.zeros(T, E, dtype=dtype, device="cuda")
    dx_slots = F.experts_bwd(dout.cuda(), y, gu, ew, b, got_dcur, dgu, dweights)
    # (equal to the last bit but for the sign of zeros, which a code has too)
    assert torch.equal(got_dcur, dcur) and torch.equal(dweights, wv.grad)
    rows = F.empty_rows(b.n_slots, H, y.device)
    N.call("usaf_hip_fp8_combine_bwd", dout.cuda().data_ptr(), y.data_ptr(), b.token_idx.data_ptr(), b.slot_w.data_ptr(),
           b.offsets.data_ptr(), b.n_slots, E, H, N.dtype_code(dtype), None, rows.q.data_ptr(), rows.s.data_ptr(),
           dweights.data_ptr(), N.stream_ptr(y.device))
    assert torch.equal(rows.q, F.quantize_rows(got_dcur).q) and torch.equal(dweights, wv.grad)
    plain = F.experts_bwd(dout.cuda(), y, gu, ew, b, None, None, torch.zeros_like(dweights))
    assert torch.equal(plain, dx_slots)
    qc = O.quantized_rows(dcur.cpu())[0]
    dgu64 = dgu.double().cpu()
    q_dgu = O.quantized_rows(dgu.cpu())[0]
    dx, dmags = torch.zeros(T, H, dtype=torch.float64), torch.zeros(T, H, dtype=torch.float64)
    for e in range(E):
        s = slice(offs[e], offs[e + 1])
        if offs[e] == offs[e + 1]:
            continue
        da = qc[s] @ wd[e]
        db = O.product_bound(qc[s], wd[e].t(), da, dtype)  # how far the kernel's d(act) may be
        dsig = sig[s] * (1 + g64[s] * (1 - sig[s]))
        ref = torch.cat([da * u64[s] * dsig, da * silu[s]], 1)
        grow = torch.cat([db * (u64[s] * dsig).abs(), db * silu[s].abs()], 1) * (1 + 4 * h)
        # at most three roundings, and the hardware exp2 / reciprocal times the conditioning of 1 + g (1 - s)
        cond = torch.cat([(da * u64[s] * sig[s]).abs() * (1 + g64[s].abs()), (da * silu[s]).abs()], 1)
        tiny = O.tiny(dtype) * torch.cat([1 + dsig.abs() * 2, 1 + da.abs()], 1)
        _within(dgu[s], ref, grow + ref.abs() * 3.1 * h + cond * 2.0 ** -19 + tiny)
        r = (q_dgu[s] @ wgu[e])
        rb = O.product_bound(q_dgu[s], wgu[e].t(), r, dtype)
        dx.index_add_(0, tok[s], r)
        dmags.index_add_(0, tok[s], rb + r.abs() * (E * 2.0 ** -24))
    _within(hv.grad, dx, dmags + dx.abs() * h + O.tiny(dtype))
    dw = torch.zeros(T, E, dtype=torch.float64)
    dw[tok, slot_e] = (dout[tok].double() * y64).sum(1)
    dm = torch.zeros(T, E, dtype=torch.float64)
    dm[tok, slot_e] = (dout[tok].double() * y64).abs().sum(1)
    _within(wv.grad, dw, dw.abs() * h + O.tiny(dtype) + H * 2.0 ** -24 * dm)
    assert dgu64.shape == (offs[-1], 2 * I)


def test_moe_block_on_8_bit_experts(F):
    """The whole block, with and without a host read, forward and backward: the same bits."""
    from usaf_amd import moe as G
    T, E, H, I, k = 50, 16, 256, 128, 2
    ew = _experts(F, E, H, I)
    hs, router = _rand(T, H, seed=1).cuda(), (_rand(E, H, seed=2) / 16).cuda()
    dout = _rand(T, H, seed=3).cuda()
    res = []
    for flag in (None, torch.zeros(1, dtype=torch.int32, device="cuda")):
        x, r = hs.clone().requires_grad_(True), router.clone().requires_grad_(True)
        out = G.moe_block(x, r, k, True, ew, overflow=flag)
        out.backward(dout)
        assert flag is None or int(flag) == 0
        res.append((out.detach(), x.grad, r.grad))
    for a, b in zip(*res):
        assert torch.equal(a, b) and bool(torch.isfinite(a).all()) and float(a.abs().max()) > 0


def test_experts_without_a_pair(F):
    from usaf_amd import moe as G
    ew = _experts(F, 4, 128, 128)
    x = _rand(3, 128).cuda().requires_grad_(True)
    w = torch.zeros(3, 4, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    out = G.routed_experts(x, w, ew)
    out.backward(torch.ones_like(out))
    assert not out.any() and not x.grad.any() and not w.grad.any()


def test_sampled_gradient_on_8_bit_experts(F):
    """A SparseGradStore gets the sampled weight gradient of 8-bit experts: positions of dgu^T hs and dcur^T act."""
    from usaf_amd import moe as G
    from usaf_amd.moe_loader import SparseGradStore
    T, E, H, I, k = 60, 4, 256, 128, 2
    ew = _experts(F, E, H, I)
    idx = {"L.gate_up_proj": torch.arange(0, E * 2 * I * H, 97), "L.down_proj": torch.arange(5, E * H * I, 101)}
    store = SparseGradStore(idx, {"L.gate_up_proj": (E, 2 * I, H), "L.down_proj": (E, H, I)}, device="cuda")
    hs, w = _rand(T, H, seed=9), _routing(T, E, k, torch.bfloat16, seed=3)
    dout = _rand(T, H, seed=11)
    x = hs.cuda().requires_grad_(True)
    out = G.routed_experts(x, w.cuda(), ew, capture=(store, "L"))
    _, gu, act, y = out.grad_fn.saved_tensors
    b = out.grad_fn.b
    gu, act, y = gu.clone(), act.double().cpu(), y.clone()
    out.backward(dout.cuda())
    offs, tok = b.offsets.tolist(), b.token_idx.long().cpu()
    slot_e = torch.repeat_interleave(torch.arange(E), torch.tensor(offs[1:]) - torch.tensor(offs[:-1]))
    dcur = (w[tok, slot_e].double()[:, None] * dout[tok].double()).bfloat16()
    dgu = torch.empty_like(gu)
    F.experts_bwd(dout.cuda(), y, gu, ew, b, None, dgu, torch.zeros(T, E, dtype=gu.dtype, device="cuda"))
    for name, left, right in (("L.gate_up_proj", dgu.double().cpu(), hs.double()[tok]), ("L.down_proj", dcur.double(), act)):
        ref = torch.stack([left[offs[e]:offs[e + 1]].t() @ right[offs[e]:offs[e + 1]] for e in range(E)]).reshape(-1)
        mag = torch.stack([left[offs[e]:offs[e + 1]].t().abs() @ right[offs[e]:offs[e + 1]].abs() for e in range(E)]).reshape(-1)
        ref, mag = ref[idx[name]], mag[idx[name]]
        # fp32 sums over at most T slots, rounded to the activations' dtype once
        _within(store.compact[name], ref, ref.abs() * O.half_step(torch.bfloat16) + 2 * T * 2.0 ** -23 * mag)


@pytest.mark.parametrize("which", [(True, True), (True, False), (False, True)])
def test_dense_weight_gradients_beside_8_bit_experts(F, which):
    """weight_params get dgu^T hs and dcur^T act of the 8-bit layer's own steps; a gradient that nobody wants is not made."""
    from usaf_amd import moe as G
    T, E, H, I, k = 60, 4, 256, 128, 2
    ew = _experts(F, E, H, I)
    wg, wd = (torch.zeros(*s, dtype=torch.float32, device="cuda").requires_grad_(r)
              for s, r in (((E, 2 * I, H), which[0]), ((E, H, I), which[1])))
    hs, w, dout = _rand(T, H, seed=9), _routing(T, E, k, torch.bfloat16, seed=3), _rand(T, H, seed=11)
    out = G.routed_experts(hs.cuda(), w.cuda(), ew, weight_params=(wg, wd))  # no gradient but the weights'
    b, gu, y = out.grad_fn.b, out.grad_fn.saved_tensors[1].clone(), out.grad_fn.saved_tensors[3].clone()
    out.backward(dout.cuda())
    offs, tok = b.offsets.tolist(), b.token_idx.long().cpu()
    slot_e = torch.repeat_interleave(torch.arange(E), torch.tensor(offs[1:]) - torch.tensor(offs[:-1]))
    dcur = (w[tok, slot_e].double()[:, None] * dout[tok].double()).bfloat16()
    dgu, act = torch.empty_like(gu), torch.empty(gu.shape[0], I, dtype=gu.dtype, device="cuda")
    F.experts_bwd(dout.cuda(), y, gu, ew, b, None, dgu, torch.zeros(T, E, dtype=gu.dtype, device="cuda"))
    F.experts_forward(F.quantize_rows(hs.cuda()), ew, b, torch.empty_like(gu), act, gu.dtype)
    for p, want, left, right in ((wg, which[0], dgu.double().cpu(), hs.double()[tok]), (wd, which[1], dcur.double(), act.double().cpu())):
        if not want:
            assert p.grad is None
            continue
        for e in range(E):
            l, r = left[offs[e]:offs[e + 1]], right[offs[e]:offs[e + 1]]
            # fp32 sums over at most T slots, stored in fp32
            _within(p.grad[e], l.t() @ r, (2 * T + 1) * 2.0 ** -23 * (l.t().abs() @ r.abs()))


def test_backward_behind_saved_tensor_hooks(F):
    """Tensors that come back from a hook in another layout, and a second backward through a kept graph: the same gradients."""
    from usaf_amd import moe as G
    ew = _experts(F, 4, 256, 128)
    hs, w, dout = _rand(60, 256, seed=9).cuda(), _routing(60, 4, 2, torch.bfloat16, seed=3).cuda(), _rand(60, 256, seed=11).cuda()

    def grads(twice=False):
        x, ww = hs.clone().requires_grad_(True), w.clone().requires_grad_(True)
        out = G.routed_experts(x, ww, ew)
        if twice:
            torch.autograd.grad(out, (x, ww), dout, retain_graph=True)
        return torch.autograd.grad(out, (x, ww), dout)

    want = grads()
    assert all(torch.equal(a, b) for a, b in zip(grads(twice=True), want))
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.t().contiguous() if t is not None and t.dim() == 2 else t,
                                                  lambda t: t.t() if t is not None and t.dim() == 2 else t):
        assert all(torch.equal(a, b) for a, b in zip(grads(), want))


def test_slots_without_a_host_read(F):
    """slot_capacity: more slots than pairs, the ones behind them unused; the same output and gradients."""
    from usaf_amd import moe as G
    T, E, H, I, k = 60, 4, 256, 128, 2
    ew = _experts(F, E, H, I)
    hs, w, dout = _rand(T, H, seed=9).cuda(), _routing(T, E, k, torch.bfloat16, seed=3).cuda(), _rand(T, H, seed=11).cuda()
    got = []
    for extra in (None, 8):
        x, ww = hs.clone().requires_grad_(True), w.clone().requires_grad_(True)
        flag = torch.zeros(1, dtype=torch.int32, device="cuda")
        kw = {} if extra is None else {"slot_capacity": T * k + extra, "overflow": flag}
        out = G.routed_experts(x, ww, ew, **kw)
        out.backward(dout)
        got.append((out.detach(), x.grad, ww.grad))
        with torch.no_grad():
            assert torch.equal(G.routed_experts(x, ww, ew, **kw), out)
        assert int(flag) == 0
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_refusals_on_the_gpu(F):
    from usaf_amd.moe import ExpertWeights, routed_experts
    t = F.Fp8Tensor.quantize(_rand(64, 128).cuda())
    x = _rand(2, 128).cuda()
    with pytest.raises(ValueError, match="on one GPU"):
        F.fp8_linear(x.cpu(), t)
    with pytest.raises(ValueError, match="do not fit"):
        F.fp8_linear(x[:, :127], t)
    with pytest.raises(TypeError, match="fp16 or bf16"):
        F.fp8_linear(x.float(), t)
    ew = _experts(F, 2, 128, 128)
    with pytest.raises(ValueError):
        routed_experts(_rand(2, 256).cuda(), torch.ones(2, 2, dtype=torch.bfloat16, device="cuda"), ew)
    with pytest.raises(NotImplementedError):
        ew.set_overlay("gate_up", torch.zeros(1, dtype=torch.int64, device="cuda"), torch.zeros(1, device="cuda"),
                       torch.bfloat16)
    with pytest.raises(TypeError, match="both"):
        ExpertWeights(ew.gate_up, torch.empty(2, 128, 128, dtype=torch.bfloat16, device="cuda"))

# every tile of the product: few to many rows, narrow and wide outputs, short and long contractions, one expert and many
TILES = [(None, 1, 33, 128), (None, 70, 33, 640), (None, 1, 2000, 1300), (None, 33, 4100, 640), (None, 4100, 200, 300),
         (None, 1000, 4100, 128), (None, 2000, 4100, 300), (None, 513, 1030, 640), (1, 2000, 130, 640), (3, 33, 4100, 640),
         (8, 200, 4100, 300), (8, 500, 4100, 128), (8, 1500, 4100, 300), (40, 33, 1030, 300), (40, 2000, 2000, 129),
         (255, 300, 130, 256), (None, 32, 9001, 1300), (8, 100, 2000, 1024)]


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("E,M,N,K", TILES)
def test_product_of_whole_numbers_on_every_tile(F, E, M, N, K, wide):
    """Exact, as test_linear_sums_whole_numbers_exactly: gathered rows, experts without a slot, slots behind the last one left."""
    dtype = DTYPES[(M + N) % 2]
    g = torch.Generator().manual_seed(M + N + K)
    n_rows = M if E is None else M // 2 + 1
    x = torch.randint(-1, 2, (n_rows, K), generator=g).to(dtype).cuda()
    w = torch.randint(-1, 2, ((E, N, K) if E else (N, K)), generator=g).float().cuda()
    out = torch.full((M, N), 333.0, dtype=dtype, device="cuda")
    rows, t = F.quantize_rows(x), F.Fp8Tensor.quantize(w)
    if E is None:
        _product(rows, t, out, wide=wide)
        assert torch.equal(out.float(), x.float() @ w.t())
        return
    ends = torch.randint(0, M - M // 8 + 1, (E,), generator=g).sort().values.tolist()
    offs = [0] + ends[:-1] + [M - M // 8]
    tok = torch.randint(0, n_rows, (M,), generator=g).to(torch.int32).cuda()
    _product(rows, t, out, torch.tensor(offs, dtype=torch.int32, device="cuda"), tok, wide=wide)
    picked = x.float()[tok.long()]
    for e in range(E):
        lo, hi = offs[e], offs[e + 1]
        assert torch.equal(out[lo:hi].float(), picked[lo:hi] @ w[e].t())
    assert bool((out[offs[-1]:] == 333).all())


@pytest.mark.parametrize("wide", [False, True])
def test_product_past_32_bits(F, wide):
    """Weights past 4 GiB and an output past 2^32 bytes: the last expert's and the last rows' places."""
    E, N, K = 40, 16384, 8192
    w = torch.ones(128, K, device="cuda")
    w[::3] = -1
    q = torch.zeros(E, N, K, dtype=torch.uint8, device="cuda")
    last = F.Fp8Tensor.quantize(w)
    q[-1, -128:] = last.q
    s = torch.full((E, N // 128, K // 128), 127, dtype=torch.uint8, device="cuda")
    s[-1, -1] = last.s[0]
    x = torch.randint(-1, 2, (5, K), generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    offs = torch.tensor([0] * E + [5], dtype=torch.int32, device="cuda")
    out = torch.empty(5, N, dtype=torch.bfloat16, device="cuda")
    _product(F.quantize_rows(x), F.Fp8Tensor(q, s, (E, N, K)), out, offs, wide=wide)
    assert torch.equal(out[:, -128:], (x.float() @ w.t()).bfloat16()) and not out[:, :-128].any()
    del q, s, out
    M, K = 140_000, 128
    w = torch.randint(-1, 2, (N, K), generator=torch.Generator().manual_seed(2)).float().cuda()
    x = torch.randint(-1, 2, (M, K), generator=torch.Generator().manual_seed(3)).bfloat16().cuda()
    out = torch.empty(M, N, dtype=torch.bfloat16, device="cuda")
    _product(F.quantize_rows(x), F.Fp8Tensor.quantize(w), out, wide=wide)
    for rows in (slice(0, 64), slice(M // 2, M // 2 + 64), slice(M - 64, M)):
        assert torch.equal(out[rows].float(), x[rows].float() @ w.t())


def test_what_is_kept_is_built_once_for_all_streams(F):
    """The transpose is built on one stream behind other work and read on another without a wait."""
    from usaf_amd.moe import Q4Tensor
    w = _rand(2048, 4096, seed=2, scale=0.1).cuda()
    x = _rand(40, 4096, seed=1).cuda()
    t, again = F.Fp8Tensor.quantize(w), F.Fp8Tensor.quantize(w)
    q4 = Q4Tensor.quantize(w.half().view(4, 512, 4096))
    dy = _rand(40, 2048, seed=3).cuda()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        busy = torch.ones(8192, 8192, device="cuda")
        for _ in range(3):
            busy = busy @ busy * 2.0 ** -13
        t.transposed()
        q4.scale_zero_by_group()
    xv = x.requires_grad_(True)
    (got,) = torch.autograd.grad(F.fp8_linear(xv, t), xv, dy)
    words = q4.scale_zero_by_group().clone()
    torch.cuda.synchronize()
    (want,) = torch.autograd.grad(F.fp8_linear(xv, again), xv, dy)
    assert torch.equal(got, want)
    assert torch.equal(words, q4.scale_zero().view(4, 512, 32).transpose(1, 2))
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            F.fp8_linear(xv, t)


def test_a_layer_tuned_and_served(F):
    """8-bit experts as they are used: prompt and gradient on the routed path of a patched block, a step of its
    norm's weight, then tokens one by one through the few-token layer, the output head in 8 bits."""
    from types import SimpleNamespace
    from usaf_amd import qwen3moe_dml as Q
    E, H, I, k, V = 8, 256, 128, 2, 1000
    ew = _experts(F, E, H, I, seed=20)
    head = F.Fp8Tensor.quantize(_rand(V, H, seed=22, scale=0.05).cuda())
    router = torch.zeros(E, H, dtype=torch.bfloat16, device="cuda")
    router[torch.arange(E), torch.arange(E)] = 1

    class Experts(torch.nn.Module):
        forward = Q.dml_qwen3_experts_forward

    class Block(torch.nn.Module):
        forward = Q.dml_qwen3_moe_block_forward

    ex, block = Experts(), Block()
    ex._usaf_q4 = {"gate_up_proj": ew.gate_up, "down_proj": ew.down}
    block.experts, block.gate = ex, SimpleNamespace(weight=router, top_k=k, norm_topk_prob=True)
    block._usaf_few_tokens = 4
    x = _rand(1, 48, H, seed=23).cuda()
    # the router reads whole numbers, so both paths route alike (no ties at the threshold)
    x[0, :, :E] = torch.stack([torch.randperm(E, generator=torch.Generator().manual_seed(i)) for i in range(48)]).to(x)
    scale = torch.ones(H, dtype=torch.bfloat16, device="cuda", requires_grad=True)

    def model(x):
        return F.fp8_linear(x * scale + block(x * scale), head)

    logits = model(x)
    assert logits.grad_fn is not None and logits.shape == (1, 48, V)
    logits.float().logsumexp(-1).sum().backward()
    assert bool(torch.isfinite(scale.grad).all()) and float(scale.grad.abs().max()) > 0
    with torch.no_grad():
        whole = model(x)
        assert torch.equal(whole, logits.detach())
        one = torch.cat([model(x[:, i:i + 1]) for i in range(48)], 1)
        four = torch.cat([model(x[:, i:i + 4]) for i in range(0, 48, 4)], 1)
    # The few-token path leaves the layer's activations unquantized.  On the routed path each of two products has operands off by
    # half a step of e4m3 at most (2^-4): a share of about 2^-4 / sqrt(3) of each term's size at random signs, so a relative error of
    # sqrt(2) * 2^-4 / sqrt(3) = 5 % of the layer's output; gate times up doubles that of its two factors.  The output head
    # quantizes both sides' inputs again, another 2 * 2^-4 / sqrt(3) = 7 % between them.  Together less than 20 %.
    ref = whole.double()
    for got in (one, four):
        assert float((got.double() - ref).norm() / ref.norm()) < 0.2


@pytest.mark.parametrize("dtype", DTYPES, ids=_ids)
@pytest.mark.parametrize("E,M,I,K", [(8, 1500, 2048, 256), (8, 500, 2176, 128), (40, 2000, 1024, 129), (200, 700, 384, 640)])
def test_gate_up_ends_in_the_activations_codes(F, E, M, I, K, dtype):
    """One launch or two: the same bits; slots behind the last one are left."""
    g = torch.Generator().manual_seed(M)
    w = F.Fp8Tensor.quantize(_rand(E, 2 * I, K, seed=E, scale=0.1).cuda())
    hs = _rand(M // 2, K, dtype=dtype, seed=K)
    hs[3, 5], hs[7, 0] = float("inf"), float("nan")
    x = F.quantize_rows(hs.cuda())
    used = M - M // 9
    ends = torch.randint(0, used + 1, (E - 1,), generator=g).sort().values.tolist()
    offs = torch.tensor([0] + ends + [used], dtype=torch.int32, device="cuda")
    tok = torch.randint(0, M // 2, (M,), generator=g).to(torch.int32).cuda()
    gu = torch.empty(M, 2 * I, dtype=dtype, device="cuda")
    _product(x, w, gu, offs, tok, wide=True)
    want, got = F.empty_rows(M, I, x.q.device), F.empty_rows(M, I, x.q.device)
    for t in (want.q, want.s, got.q, got.s):
        t.fill_(77)
    N.call("usaf_hip_fp8_swiglu", gu.data_ptr(), M, I, N.dtype_code(dtype), offs[-1:].data_ptr(), None, want.q.data_ptr(),
           want.s.data_ptr(), N.stream_ptr(x.q.device))
    N.call("usaf_hip_fp8_gate_up", x.q.data_ptr(), x.s.data_ptr(), x.q.shape[0], tok.data_ptr(), M, w.q.data_ptr(),
           w.s.data_ptr(), offs.data_ptr(), E, I, K, N.dtype_code(dtype), got.q.data_ptr(), got.s.data_ptr(),
           N.stream_ptr(x.q.device))
    assert torch.equal(got.q, want.q) and torch.equal(got.s, want.s)


def test_experts_without_a_backward_keep_nothing(F):
    """The same bits with and without a gradient in sight."""
    from usaf_amd import moe as G
    ew = _experts(F, 4, 256, 2048, seed=30)  # (gate and up in one launch)
    hs, w = _rand(600, 256, seed=31).cuda(), _routing(600, 4, 2, torch.bfloat16, seed=32).cuda()
    want = G.routed_experts(hs.clone().requires_grad_(True), w, ew).detach()
    assert torch.equal(G.routed_experts(hs, w, ew), want)
    with torch.no_grad():
        assert torch.equal(G.routed_experts(hs.clone().requires_grad_(True), w, ew), want)


@pytest.mark.parametrize("rows", [3, 50])
def test_linear_under_a_trace_and_a_tangent(F, rows):
    """A trace replays the product, not the memory it was written to; a forward-mode derivative is refused."""
    from torch.autograd import forward_ad
    t = F.Fp8Tensor.quantize(_rand(200, 384, seed=2, scale=0.1).cuda())
    x, other = _rand(rows, 384, seed=1).cuda(), _rand(rows, 384, seed=2).cuda()
    with torch.no_grad():
        traced = torch.jit.trace(lambda v: F.fp8_linear(v, t) * 2, (x,))
        for v in (other, x):
            assert torch.equal(traced(v), F.fp8_linear(v, t) * 2)
    with forward_ad.dual_level():
        with pytest.raises((NotImplementedError, RuntimeError), match="forward"):
            F.fp8_linear(forward_ad.make_dual(x, x), t)
        assert torch.equal(F.fp8_linear(x, t), F.fp8_linear(x.clone(), t))
