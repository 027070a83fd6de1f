"""The 8-bit and few-token layers at the sizes of whole models' layers, and at the few-token layer's limits, against 64 bits.

Every case is run twice and has to give the same bits."""
import pytest
import torch

import fp8_oracle as O

pytestmark = pytest.mark.gpu
LAYERS = {  # experts, hidden, intermediate, experts of a token
    "qwen3-30b-a3b": (128, 2048, 768, 8),
    "olmoe-1b-7b": (64, 2048, 1024, 8),
    "mixtral-8x7b": (8, 4096, 14336, 2),
}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rand(*shape, dtype=torch.bfloat16, seed=0, scale=1.0):
    return (torch.randn(*shape, device="cuda", generator=_gen(seed)) * scale).to(dtype)


def _weights(fmt, E, R, C, seed):
    """A weight of about 0.02 from random codes."""
    from usaf_amd.fp8 import Fp8Tensor
    from usaf_amd.moe import Q4Tensor
    g, dev = _gen(seed), "cuda"
    if fmt == "fp8":
        q = torch.empty(E, R, C, dtype=torch.uint8, device=dev)
        for e in range(E):
            q[e] = (torch.randn(R, C, device=dev, generator=g) * 96).clamp_(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
        s = torch.randint(127 - 13, 127 - 11, (E, R // 128, C // 128), device=dev, generator=g).to(torch.uint8)
        return Fp8Tensor(q, s, (E, R, C))
    n = E * R * C // 128
    q = torch.randint(0, 256, (n, 64), dtype=torch.uint8, device=dev, generator=g).view(torch.int8)
    s = (0.0035 + 0.002 * torch.rand(n, device=dev, generator=g)).half()
    z = (-7.5 * s.float() * (0.9 + 0.2 * torch.rand(n, device=dev, generator=g))).half()
    return Q4Tensor(q, s, z, torch.Size((E, R, C)))


def _layer(fmt, E, H, I, seed=0):
    from usaf_amd.moe import ExpertWeights
    return ExpertWeights(_weights(fmt, E, 2 * I, H, seed), _weights(fmt, E, H, I, seed + 1))


def _matrix(t, e):
    """Matrix e of a weight in 64 bits."""
    _, R, C = t.shape
    if hasattr(t, "z"):
        n = R * C // 128
        q, s, z = (v[e * n:(e + 1) * n] for v in (t.q, t.s, t.z))
        b = q.view(torch.uint8)
        codes = torch.stack([b & 15, b >> 4], -1).reshape(n, 128).double()
        return (codes * s.double()[:, None] + z.double()[:, None]).view(R, C)
    return O.values(t.q[e], t.s[e], (R, C))


# ---- few tokens ------------------------------------------------------------------

def _check_few(ew, k, T, dtype, norm, seed):
    from usaf_amd.few import few_token_block
    E, H, I = ew.E, ew.H, ew.I
    x, router = _rand(T, H, dtype=dtype, seed=seed), _rand(E, H, dtype=dtype, seed=seed + 1, scale=1.5 / H ** 0.5)
    with torch.no_grad():
        out = few_token_block(x, router, k, norm, ew)
        assert torch.equal(few_token_block(x, router, k, norm, ew), out)
    logits = x.double() @ router.double().t()
    order = torch.argsort(-logits, dim=1, stable=True)[:, :k]
    p = torch.softmax(logits, 1)
    w = torch.zeros_like(p).scatter_(1, order, p.gather(1, order))
    w = w / w.sum(1, keepdim=True) if norm else w
    ref = torch.zeros(T, H, dtype=torch.float64, device="cuda")
    for e in range(E):
        rows = w[:, e].nonzero().reshape(-1)
        if rows.numel():
            g, u = (x[rows].double() @ _matrix(ew.gate_up, e).t()).split(I, 1)
            ref[rows] += w[rows, e:e + 1] * ((g * torch.sigmoid(g) * u) @ _matrix(ew.down, e).t())
    # By a token's norm: the output's rounding is at most half a step; the gated activations' roundings, half a step each at
    # signs of their own, add about as much at most; fp32 sums are far below.  Three half steps leave the second a factor of two.
    rel = (out.double() - ref).norm(dim=1) / ref.norm(dim=1)
    assert float(rel.max()) <= 3 * O.half_step(dtype), rel.max()


@pytest.mark.parametrize("fmt", ["q4", "fp8"])
@pytest.mark.parametrize("name", LAYERS)
def test_few_tokens(name, fmt):
    E, H, I, k = LAYERS[name]
    ew = _layer(fmt, E, H, I)
    for T, dtype in ((1, torch.bfloat16), (2, torch.float16), (7, torch.float16), (24, torch.bfloat16), (32, torch.bfloat16)):
        _check_few(ew, k, T, dtype, T % 2 == 0, seed=T)


@pytest.mark.parametrize("fmt", ["q4", "fp8"])
@pytest.mark.parametrize("E,H,I,k", [(2, 16384, 128, 1), (2, 128, 65536, 1), (2, 16384, 65536, 2), (256, 128, 256, 16)])
def test_few_tokens_at_the_limits(E, H, I, k, fmt):
    """The widest layers: one or two parts of a column tile, the longest rows of the buffers, the most steps of a wave."""
    ew = _layer(fmt, E, H, I)
    for T, dtype in ((1, torch.bfloat16), (3, torch.float16), (32, torch.bfloat16)):
        _check_few(ew, k, T, dtype, T == 3, seed=T)


# ---- routed 8-bit experts --------------------------------------------------------

def _within(what, got, ref, bound):
    off = (got.double() - ref).abs() - bound
    assert float(off.max()) <= 0, f"{what}: {float(off.max())} past the bound"


@pytest.mark.parametrize("name,T,dtype", [("qwen3-30b-a3b", 256, torch.bfloat16), ("qwen3-30b-a3b", 2048, torch.float16),
                                          ("olmoe-1b-7b", 700, torch.float16), ("mixtral-8x7b", 300, torch.bfloat16),
                                          ("mixtral-8x7b", 40, torch.float16)])
def test_routed_8_bit_experts(name, T, dtype):
    """Every step of the pass and its backward against 64 bits of what that step was given."""
    from usaf_amd import fp8 as F, moe as G
    E, H, I, k = LAYERS[name]
    ew = _layer("fp8", E, H, I, seed=3)
    hs, dout = _rand(T, H, dtype=dtype, seed=9), _rand(T, H, dtype=dtype, seed=11)
    p = torch.softmax(torch.randn(T, E, device="cuda", generator=_gen(12)) - torch.arange(1, E + 1, device="cuda").log(), -1)
    top = p.topk(k, -1)
    w = torch.zeros_like(p).scatter_(1, top.indices, top.values / top.values.sum(-1, keepdim=True)).to(dtype)

    def run():
        hv, wv = hs.clone().requires_grad_(True), w.clone().requires_grad_(True)
        out = G.routed_experts(hv, wv, ew)
        fn = out.grad_fn
        saved = fn.saved_tensors
        out.backward(dout, retain_graph=True)
        return out.detach(), hv.grad, wv.grad, saved, fn.b

    out, dx, dw, (_, gu, _, y), b = run()
    assert all(torch.equal(a, c) for a, c in zip(run()[:3], (out, dx, dw)))
    with torch.no_grad():
        assert torch.equal(G.routed_experts(hs, w, ew), out)
    act = torch.empty(b.n_slots, I, dtype=dtype, device="cuda")
    assert torch.equal(F.experts_forward(F.quantize_rows(hs), ew, b, torch.empty_like(gu), act, dtype), y)
    dcur, dgu = torch.empty_like(y), torch.empty_like(gu)
    dx_slots = F.experts_bwd(dout, y, gu, ew, b, dcur, dgu, torch.zeros(T, E, dtype=dtype, device="cuda"))
    offs, tok, h = b.offsets.tolist(), b.token_idx.long(), O.half_step(dtype)
    sums, mags = torch.zeros(T, H, dtype=torch.float64, device="cuda"), torch.zeros(T, H, dtype=torch.float64, device="cuda")
    dsums, dmags = torch.zeros_like(sums), torch.zeros_like(sums)
    for e in range(E):
        s = slice(offs[e], offs[e + 1])
        if offs[e] == offs[e + 1]:
            continue
        t, we = tok[s], w[tok[s], e].double()[:, None]
        wgu, wd = _matrix(ew.gate_up, e), _matrix(ew.down, e)
        a = O.quantized_rows(hs[t])[0]
        ref = a @ wgu.t()
        _within("gate, up", gu[s], ref, O.wide_bound(a, wgu, ref, dtype))
        g, u = gu[s].double().split(I, 1)
        sig = torch.sigmoid(g)
        silu = g * sig
        # silu and its product are rounded one behind the other; the hardware's exp2 and reciprocal are good to about 2^-22
        _within("activation", act[s], silu * u, (silu * u).abs() * (2.01 * h + 2.0 ** -20) + O.tiny(dtype) * (1 + u.abs()))
        a = O.quantized_rows(act[s])[0]
        ref = a @ wd.t()
        _within("down", y[s], ref, O.product_bound(a, wd, ref, dtype))
        sums.index_add_(0, t, we * y[s].double())
        mags.index_add_(0, t, (we * y[s].double()).abs())
        ref = (dout[t].double() * y[s].double()).sum(1)
        mag = (dout[t].double() * y[s].double()).abs().sum(1)
        _within("d(weights)", dw[t, e], ref, ref.abs() * h + O.tiny(dtype) + H * 2.0 ** -24 * mag)
        assert torch.equal(dcur[s], (we * dout[t].double()).to(dtype))
        a = O.quantized_rows(dcur[s])[0]
        da = a @ wd
        db = O.wide_bound(a, wd.t(), da, dtype)
        dsig = sig * (1 + g * (1 - sig))
        ref = torch.cat([da * u * dsig, da * silu], 1)
        grow = torch.cat([db * (u * dsig).abs(), db * silu.abs()], 1) * (1 + 4 * h)
        # at most three roundings, and the hardware's functions times the conditioning of 1 + g (1 - s)
        cond = torch.cat([(da * u * sig).abs() * (1 + g.abs()), (da * silu).abs()], 1)
        tiny = O.tiny(dtype) * torch.cat([1 + dsig.abs() * 2, 1 + da.abs()], 1)
        _within("d(gate, up)", dgu[s], ref, grow + ref.abs() * 3.1 * h + cond * 2.0 ** -19 + tiny)
        a = O.quantized_rows(dgu[s])[0]
        ref = a @ wgu
        _within("d(hidden) of a slot", dx_slots[s], ref, O.product_bound(a, wgu.t(), ref, dtype))
        dsums.index_add_(0, t, dx_slots[s].double())
        dmags.index_add_(0, t, dx_slots[s].double().abs())
    _within("output", out, sums, sums.abs() * h + O.tiny(dtype) + (E + 1) * 2.0 ** -24 * mags)
    _within("d(hidden)", dx, dsums, dsums.abs() * h + O.tiny(dtype) + (E + 1) * 2.0 ** -24 * dmags)
