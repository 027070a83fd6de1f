"""The gated projection on the GPU against the 64-bit oracle: activation, what is kept for the backward, gradients."""
import pytest
import torch

import fp8_oracle as F8
import linear_oracle as O
from usaf_amd import _native as N

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]
# tokens, intermediate, hidden: one row to many, columns that fill no 8, no 16, no 128
Q4_SIZES = [(1, 1, 128), (1, 128, 256), (2, 5, 128), (9, 130, 384), (31, 257, 640), (33, 128, 256), (64, 96, 384), (65, 711, 256),
            (130, 255, 512), (300, 384, 512), (511, 40, 256), (513, 300, 896), (1030, 264, 384),
            (8, 33, 4096), (16, 300, 2048), (1, 40, 14336), (5, 1000, 1920), (1, 9000, 256)]
DENSE_SIZES = [(1, 1, 1), (1, 128, 64), (2, 5, 127), (9, 130, 129), (31, 257, 640), (33, 128, 100), (65, 711, 200),
               (130, 255, 512), (300, 384, 512), (257, 70, 1000), (600, 520, 192)]


def _ids(d):
    return str(d).replace("torch.", "")


@pytest.fixture(scope="module")
def G():
    from usaf_amd import gated
    return gated


def _q4(rows, k, seed, scale=0.03):
    from usaf_amd.moe import Q4Tensor
    parts = O.codes(rows, k, seed, scale)
    return Q4Tensor(*(t.cuda() for t in parts), torch.Size((rows, k))), parts


def _rand(*shape, dtype, seed=1, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def _kept(G, x, w, checkpoint):
    """What a forward keeps: float64 gate and up, with their scales (checkpoints)."""
    from usaf_amd.q4 import rows_of
    inter = w.shape[0] // 2
    weight = w if not isinstance(w, torch.Tensor) else G._dense(w.detach())
    act, kept, scales = G._forward(rows_of(x.detach(), x.shape[1]), weight, checkpoint, True)
    if checkpoint is None:
        v = kept.double().cpu()
        return act, v[:, 0, :inter], v[:, 1, :inter], None
    s = torch.exp2(scales.cpu().double() - 127)
    v = kept.cpu().view(torch.float8_e4m3fn).double() * s.repeat_interleave(128, -1)
    assert not v[:, :, inter:].any()  # codes behind the last column are zeros
    return act, v[:, 0, :inter], v[:, 1, :inter], s


def _check(G, x, w, w64, checkpoint, dtype, dact):
    (g, off_g), (u, off_u), (ref, off) = O.gated(x.detach().double().cpu(), w64)
    leaves = [x] + ([w] if isinstance(w, torch.Tensor) else [])
    act = G.gated_linear(x, w, checkpoint=checkpoint)
    assert act.dtype == dtype
    O.within(act, ref, O.rounded(ref, off, dtype), "act")
    again, kg, ku, s = _kept(G, x, w, checkpoint)
    assert torch.equal(again, act)
    for i, (name, got, v, o) in enumerate((("gate", kg, g, off_g), ("up", ku, u, off_u))):
        if checkpoint is None:
            O.within(got, v, O.rounded(v, o, dtype), name)
            continue
        # the scale is the oracle's for a largest magnitude within the sum's error; a code is at most half a step off
        pad = (0, -v.shape[1] % 128)
        blocks = [torch.nn.functional.pad(t, pad).view(v.shape[0], -1, 128) for t in (v.abs(), o)]
        top = blocks[0].amax(-1), blocks[1].amax(-1)
        e = torch.log2(s[:, i]).long()
        assert bool((F8.exponent((top[0] - top[1]).clamp_min(0)) <= e).all())
        assert bool((e <= F8.exponent(top[0] + top[1])).all())
        step = s[:, i].repeat_interleave(128, -1)[:, :v.shape[1]]
        O.within(got, v, torch.maximum((v.abs() + o) * 2.0 ** -4, step * 2.0 ** -10) * (1 + 2.0 ** -20) + o, name)
    act.backward(dact.cuda())
    (dg, od_g), (du, od_u) = O.gated_grads(dact.double(), kg, ku)
    dgu, od = torch.cat([dg, du], 1), torch.cat([od_g, od_u], 1)
    od = O.rounded(dgu, od, dtype)
    ref, off = O.product(dgu, w64.t().contiguous())
    O.within(x.grad, ref, O.rounded(ref, off + od @ w64.abs(), dtype), "dx")
    # the roundings of dG and dU and of dx add up like random ones, at most half a step each
    if ref.numel() >= 4096:
        assert O.rms_off(x.grad, ref) <= 1.5 * F8.half_step(dtype)
    if len(leaves) > 1:
        xt = x.detach().double().cpu().t().contiguous()
        ref, off = O.product(dgu.t().contiguous(), xt)
        O.within(w.grad, ref, O.rounded(ref, off + od.t() @ xt.abs().t(), dtype), "dw")
        if ref.numel() >= 4096:
            assert O.rms_off(w.grad, ref) <= 1.5 * F8.half_step(dtype)
    return act


@pytest.mark.parametrize("checkpoint", [None, "fp8"])
@pytest.mark.parametrize("dtype", DTYPES, ids=_ids)
@pytest.mark.parametrize("m,inter,k", Q4_SIZES)
def test_4bit_weights(G, m, inter, k, dtype, checkpoint):
    w, parts = _q4(2 * inter, k, m + inter)
    x = _rand(m, k, dtype=dtype).cuda().requires_grad_()
    w64 = O.weight(*parts, 2 * inter, k, dtype)
    act = _check(G, x, w, w64, checkpoint, dtype, _rand(m, inter, dtype=dtype, seed=2))
    with torch.no_grad():
        plain = G.gated_linear(x, w, checkpoint=checkpoint)
    # (a pass without a gradient may take other tiles, whose sums come in another order: both are within the sums' bound)
    O.within(plain, *(lambda r, o: (r, O.rounded(r, o, dtype)))(*O.gated(x.detach().double().cpu(), w64)[2]), "without a gradient")


@pytest.mark.parametrize("checkpoint", [None, "fp8"])
@pytest.mark.parametrize("dtype", DTYPES, ids=_ids)
@pytest.mark.parametrize("m,inter,k", DENSE_SIZES)
def test_16bit_weights(G, m, inter, k, dtype, checkpoint):
    w = _rand(2 * inter, k, dtype=dtype, seed=5, scale=0.1)
    x = _rand(m, k, dtype=dtype).cuda().requires_grad_()
    _check(G, x, w.cuda().requires_grad_(), w.double(), checkpoint, dtype, _rand(m, inter, dtype=dtype, seed=2))


def test_which_gradients_are_wanted(G):
    x0, w0, d = (_rand(*s, dtype=torch.bfloat16, seed=i).cuda() for i, s in enumerate([(50, 192), (260, 192), (50, 130)]))
    both = [x0.clone().requires_grad_(), w0.clone().requires_grad_()]
    G.gated_linear(*both).backward(d)
    x = x0.clone().requires_grad_()
    G.gated_linear(x, w0).backward(d)
    w = w0.clone().requires_grad_()
    G.gated_linear(x0, w).backward(d)
    assert torch.equal(x.grad, both[0].grad) and torch.equal(w.grad, both[1].grad)
    # a frozen weight in other places and orders
    t = w0.t().contiguous().t()
    shifted = torch.empty(260 * 192 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(260, 192).copy_(w0)
    ref = G.gated_linear(x0, w0)
    assert torch.equal(G.gated_linear(x0, t), ref) and torch.equal(G.gated_linear(x0, shifted), ref)
    w = t.detach().requires_grad_()
    G.gated_linear(x0, w).backward(d)
    assert torch.equal(w.grad, both[1].grad)


def test_what_is_kept(G):
    """Bytes that a graph holds: 4 I a token, 2 I (1 + 1/128) with checkpoints, nothing without a gradient."""
    w, _ = _q4(1024, 256, 0)
    x = _rand(64, 256, dtype=torch.bfloat16).cuda().requires_grad_()
    sizes = {}
    for checkpoint in (None, "fp8"):
        held = []
        with torch.autograd.graph.saved_tensors_hooks(lambda t: (held.append(t.numel() * t.element_size()), t)[1], lambda t: t):
            G.gated_linear(x, w, checkpoint=checkpoint)
        sizes[checkpoint] = sum(held)
    assert sizes == {None: 64 * 4 * 512, "fp8": 64 * (2 * 512 + 2 * 4)}
    # hooks that give back tensors in another order
    ref = torch.autograd.grad(G.gated_linear(x, w, checkpoint="fp8").sum(), x)[0]
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.cuda().transpose(0, -1).contiguous().transpose(0, -1)):
        out = G.gated_linear(x, w, checkpoint="fp8")
    assert torch.equal(torch.autograd.grad(out.sum(), x)[0], ref)


def test_shapes_strides_and_empty_calls(G):
    w, _ = _q4(260, 256, 3)
    x = _rand(24, 256, dtype=torch.float16).cuda()
    y = G.gated_linear(x, w)
    assert torch.equal(G.gated_linear(x.view(2, 3, 4, 256), w), y.view(2, 3, 4, 130))
    assert torch.equal(G.gated_linear(x[0], w), G.gated_linear(x[:1], w)[0])
    wide = torch.zeros(24, 301, dtype=torch.float16, device="cuda")
    for first in (0, 3):
        wide[:, first:first + 256] = x
        assert torch.equal(G.gated_linear(wide[:, first:first + 256], w), y)
    assert torch.equal(G.gated_linear(x.flip(0), w), y.flip(0))
    assert torch.equal(G.gated_linear(x[:1].expand(24, 256), w), y[:1].expand(24, 130))
    xg = x.view(4, 6, 256).clone().requires_grad_()
    G.gated_linear(xg, w).sum().backward()
    x1 = x.clone().requires_grad_()
    G.gated_linear(x1, w).backward(torch.ones(130, 24, dtype=torch.float16, device="cuda").t())
    assert torch.equal(xg.grad.view(24, 256), x1.grad)
    for shape in [(0, 256), (2, 0, 256)]:
        for weight in (w, _rand(260, 256, dtype=torch.float16).cuda().requires_grad_()):
            for checkpoint in (None, "fp8"):
                e = torch.zeros(*shape, dtype=torch.float16, device="cuda", requires_grad=True)
                out = G.gated_linear(e, weight, checkpoint=checkpoint)
                assert out.shape == (*shape[:-1], 130)
                out.sum().backward()
                assert e.grad.shape == e.shape
                if isinstance(weight, torch.Tensor):
                    assert not weight.grad.any()
                    weight.grad = None


@pytest.mark.parametrize("checkpoint", [None, "fp8"])
def test_rows_that_are_not_finite_stay_alone(G, checkpoint):
    w, _ = _q4(2 * 200, 256, 3)
    for m in (3, 70, 600):
        d = _rand(m, 200, dtype=torch.bfloat16, seed=4).cuda()
        x = _rand(m, 256, dtype=torch.bfloat16).cuda().requires_grad_()
        y = G.gated_linear(x, w, checkpoint=checkpoint)
        y.backward(d)
        bad = x.detach().clone()
        bad[m // 2, 9] = float("nan")
        bad.requires_grad_()
        z = G.gated_linear(bad, w, checkpoint=checkpoint)
        z.backward(d)
        keep = (torch.arange(m) != m // 2).cuda()
        assert bool(torch.isnan(z[m // 2]).all()) and bool(torch.isnan(bad.grad[m // 2]).all())
        assert torch.equal(z[keep], y[keep]) and torch.equal(bad.grad[keep], x.grad[keep])


def test_large_gates(G):
    """silu and its derivative at their ends: -x where gate is far below zero, x above."""
    k, inter = 128, 64
    w = torch.zeros(2 * inter, k, dtype=torch.bfloat16)
    w[:inter, 0] = torch.linspace(-300, 300, inter).bfloat16()
    w[inter:, 1] = 1
    x = torch.zeros(2, k, dtype=torch.bfloat16)
    x[:, 0], x[:, 1] = torch.tensor([1.0, -1.0]).bfloat16(), 2
    xg = x.cuda().requires_grad_()
    for checkpoint in (None, "fp8"):
        xg.grad = None
        out = _check(G, xg, w.cuda().requires_grad_(), w.double(), checkpoint, torch.bfloat16, torch.ones(2, inter).bfloat16())
        assert bool(torch.isfinite(out).all()) and bool(torch.isfinite(xg.grad).all())


def test_in_a_graph_and_on_streams(G):
    w, _ = _q4(2 * 320, 640, 1)
    wd = _rand(2 * 320, 640, dtype=torch.bfloat16, scale=0.1).cuda()
    for weight in (w, wd):
        for m in (1, 40, 600):
            x = _rand(m, 640, dtype=torch.bfloat16).cuda()
            with torch.no_grad():
                G.gated_linear(x, weight)
                torch.cuda.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    y = G.gated_linear(x, weight)
                for seed in range(3):
                    x.copy_(_rand(m, 640, dtype=torch.bfloat16, seed=seed + 10))
                    want = G.gated_linear(x, weight)
                    graph.replay()
                    torch.cuda.synchronize()
                    assert torch.equal(y, want)
    graph = torch.cuda.CUDAGraph()
    x = _rand(4, 640, dtype=torch.bfloat16).cuda()
    with torch.cuda.graph(graph):
        z = x * 2
        with pytest.raises(RuntimeError, match="captured"):
            G.gated_linear(x.requires_grad_(), w)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(z, x.detach() * 2)
    # forward and backward on two streams at once
    def step(seed):
        leaf = _rand(300, 640, dtype=torch.bfloat16, seed=seed).cuda().requires_grad_()
        G.gated_linear(leaf, w, checkpoint="fp8").float().pow(2).sum().backward()
        return leaf.grad
    ref = [step(s) for s in range(4)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for s in range(4):
        with torch.cuda.stream(streams[s % 2]):
            got.append(step(s))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(ref, got))


def test_second_derivatives_and_traces(G):
    w, _ = _q4(64, 128, 0)
    x = _rand(3, 128, dtype=torch.float16).cuda().requires_grad_()
    with pytest.raises(RuntimeError, match="second"):
        torch.autograd.grad(G.gated_linear(x, w).sum(), x, create_graph=True)
    from torch.autograd import forward_ad
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x.detach(), torch.ones_like(x))
        with pytest.raises((RuntimeError, NotImplementedError)):
            G.gated_linear(dual, w)
    plain = x.detach()
    traced = torch.jit.trace(lambda t: G.gated_linear(t, w), (plain,), check_trace=False)
    assert torch.equal(traced(plain * 2), G.gated_linear(plain * 2, w))


@pytest.mark.parametrize("m", [1, 12, 200, 700])
def test_a_feed_forward_layer(G, m):
    """gate and up, activation, down: a dense layer on 4-bit weights, forward and backward, against the routed layer's only
    expert with the same weights, whose 16-bit steps in between round more."""
    from usaf_amd.moe import ExpertWeights, Q4Tensor, routed_experts
    from usaf_amd.q4 import q4_linear
    hidden, inter, dtype = 256, 384, torch.bfloat16
    gu, parts = _q4(2 * inter, hidden, 1)
    dn, parts_d = _q4(hidden, inter, 2)
    x, d = (_rand(m, hidden, dtype=dtype, seed=s).cuda() for s in (1, 2))
    xg = x.clone().requires_grad_()
    out = q4_linear(G.gated_linear(xg, gu, checkpoint="fp8"), dn)
    out.backward(d)
    w, wd = O.weight(*parts, 2 * inter, hidden, dtype), O.weight(*parts_d, hidden, inter, dtype)
    (g, _), (u, _), (act, _) = O.gated(x.double().cpu(), w)
    ref = act @ wd.t()
    assert O.rms_off(out, ref) <= 2 * F8.half_step(dtype)  # two roundings
    ew = ExpertWeights(Q4Tensor(gu.q, gu.s, gu.z, torch.Size((1, 2 * inter, hidden))),
                       Q4Tensor(dn.q, dn.s, dn.z, torch.Size((1, hidden, inter))))
    xr = x.clone().requires_grad_()
    routed = routed_experts(xr, torch.ones(m, 1, dtype=dtype, device="cuda"), ew)
    routed.backward(d)
    assert O.rms_off(out, routed.detach().double().cpu()) <= 6 * F8.half_step(dtype)  # its six roundings
    # the checkpoints' 4 significant bits: at most 2^-4 of gate and of up each, in dG = d u s (1 + g (1 - s)) and dU = d g s
    assert O.rms_off(xg.grad, xr.grad.double().cpu()) <= 3 * 2.0 ** -4


def test_workspaces_that_are_too_small(G):
    x, w = _rand(40, 100, dtype=torch.float16).cuda(), _rand(64, 100, dtype=torch.float16).cuda()
    act = torch.empty(40, 32, dtype=torch.float16, device="cuda")
    need = N.load().usaf_hip_gated_ws_bytes(40, 32, 100, 0, 0)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    for size in (0, need - 1):
        with pytest.raises(ValueError, match="workspace"):
            N.call("usaf_hip_gated_fwd", x.data_ptr(), N.F16, 40, 100, 100, None, None, w.data_ptr(), 32, act.data_ptr(), None,
                   None, ws.data_ptr(), size, N.stream_ptr(x.device))
