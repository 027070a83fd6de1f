"""The few-token MoE layer on 4-bit and 8-bit experts against the layer's definition in 64 bits."""
import pytest
import torch

import fp8_oracle as O

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]


def _ids(d):
    return str(d).replace("torch.", "")


@pytest.fixture(scope="module")
def B():
    from usaf_amd import few
    return few


def _rand(*shape, dtype=torch.bfloat16, seed=0, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def _experts(fmt, gate_up, down):
    """ExpertWeights from float weights, and the values they stand for in 64 bits."""
    from usaf_amd.fp8 import Fp8Tensor
    from usaf_amd.moe import ExpertWeights, Q4Tensor
    made, vals = [], []
    for w in (gate_up, down):
        if fmt == "fp8":
            t = Fp8Tensor.quantize(w.cuda())
            vals.append(O.values(t.q.cpu(), t.s.cpu(), w.shape))
        else:
            t = Q4Tensor.quantize(w.half().cuda())
            b = t.q.cpu().view(torch.uint8)
            codes = torch.stack([b & 15, b >> 4], -1).reshape(-1, 128).double()
            vals.append((codes * t.s.cpu().double()[:, None] + t.z.cpu().double()[:, None]).view(w.shape))
        made.append(t)
    return ExpertWeights(*made), vals


def _random_experts(fmt, E, H, I, seed=0):
    return _experts(fmt, _rand(E, 2 * I, H, dtype=torch.float32, seed=seed, scale=0.05),
                    _rand(E, H, I, dtype=torch.float32, seed=seed + 1, scale=0.05))


def _route(x, router, k, norm):
    """[T, E] weights in 64 bits: the k largest logits, the lowest expert of equal ones."""
    l = x.double() @ router.double().t()
    order = torch.argsort(-l, dim=1, stable=True)[:, :k]
    p = torch.softmax(l, 1)
    w = torch.zeros_like(p).scatter_(1, order, p.gather(1, order))
    return w / w.sum(1, keepdim=True) if norm else w


def _layer(x, w, vals):
    """The layer in 64 bits, the gated activation not rounded."""
    gu, dn = vals
    out = torch.zeros(x.shape, dtype=torch.float64)
    I = dn.shape[2]
    for e in range(gu.shape[0]):
        rows = (w[:, e] != 0).nonzero().reshape(-1)
        if rows.numel():
            g, u = (x[rows].double() @ gu[e].t()).split(I, 1)
            out[rows] += w[rows, e:e + 1] * ((g * torch.sigmoid(g) * u) @ dn[e].t())
    return out


def _check(out, ref, dtype):
    """Each token's row, by its norm: the output's rounding is at most half a step; the gated activations'
    roundings, half a step each with signs of their own, add at most about as much; fp32 sums are far below.  Three half
    steps leave the second a factor of two."""
    out, ref = out.double().cpu(), ref.view(out.shape)
    assert bool(torch.isfinite(out).all())
    rel = (out - ref).norm(dim=-1) / ref.norm(dim=-1)
    assert float(rel.max()) <= 3 * O.half_step(dtype), rel.max()


SHAPES = [  # E, H, I, k
    (8, 256, 128, 2), (1, 128, 128, 1), (5, 384, 256, 5), (64, 128, 384, 8), (256, 128, 128, 16), (130, 640, 128, 3),
    (3, 1024, 512, 1),
]


@pytest.mark.parametrize("dtype", DTYPES, ids=_ids)
@pytest.mark.parametrize("fmt", ["q4", "fp8"])
@pytest.mark.parametrize("T", [1, 2, 9, 31, 32])
@pytest.mark.parametrize("E,H,I,k", SHAPES)
def test_layer(B, E, H, I, k, T, fmt, dtype):
    ew, vals = _random_experts(fmt, E, H, I)
    x, router = _rand(T, H, dtype=dtype, seed=T), _rand(E, H, dtype=dtype, seed=5, scale=1.5 / H ** 0.5)
    norm = T % 2 == 1
    out = B.few_token_block(x.cuda(), router.cuda(), k, norm, ew)
    _check(out, _layer(x, _route(x, router, k, norm), vals), dtype)


@pytest.mark.parametrize("dtype", DTYPES, ids=_ids)
@pytest.mark.parametrize("fmt", ["q4", "fp8"])
def test_whole_numbers_come_out_exactly(B, fmt, dtype):
    """Gates of 32 (silu(32) = 32 in fp32), whole weights, equal routing weights: no step rounds, so a code, scale, token or
    column at a wrong place shows."""
    E, H, I, k, T = 6, 256, 256, 2, 32
    g = torch.Generator().manual_seed(1)
    # 4-bit: scale 1 and zero -8 need the codes' whole range -8 .. 7 in each group
    gu = torch.zeros(E, 2 * I, H)
    gu[:, :I, 1] = 4
    gu[:, I:] = torch.randint(-1, 2, (E, I, H), generator=g).float() * (torch.rand(E, I, H, generator=g) < 0.02)
    gu[:, :, 126], gu[:, :, 127], gu[:, :, 254], gu[:, :, 255] = -8, 7, -8, 7
    dn = torch.randint(-1, 2, (E, H, I), generator=g).float() * (torch.rand(E, H, I, generator=g) < 0.05)
    dn[:, :, 0], dn[:, :, 1], dn[:, :, 128], dn[:, :, 129] = -8, 7, -8, 7
    gu[:, I:, :2] = 0
    x = torch.randint(-2, 3, (T, H), generator=g).float()
    x[:, 1] = 8
    x[:, 126] = x[:, 127] = x[:, 254] = x[:, 255] = 0
    x[:, 0] = 0
    router = torch.zeros(E, H)
    x[:, 2:2 + E] = 0
    gu[:, I:, 2:2 + E] = 0
    for t in range(T):  # two experts a token with equal logits, far above the rest
        a, b = t % E, (t * 3 + 1) % E if (t * 3 + 1) % E != t % E else (t + 1) % E
        x[t, 2 + a] = x[t, 2 + b] = 4
    router[torch.arange(E), 2 + torch.arange(E)] = 64
    for e in range(E):  # down rows 0, 1, 128, 129 hold the range's ends: their activations are zero
        gu[e, I + torch.tensor([0, 1, 128, 129])] = 0
        gu[e, I + torch.tensor([0, 1, 128, 129]), 126] = -8
        gu[e, I + torch.tensor([0, 1, 128, 129]), 127] = 7
        gu[e, I + torch.tensor([0, 1, 128, 129]), 254] = -8
        gu[e, I + torch.tensor([0, 1, 128, 129]), 255] = 7
    ew, vals = _experts(fmt, gu, dn)
    assert torch.equal(vals[0], gu.double()) and torch.equal(vals[1], dn.double())
    w = _route(x, router, k, True)
    assert set(w.unique().tolist()) == {0.0, 0.5}
    ref = _layer(x.to(dtype), w, vals).round()  # 64 bits tell silu(32) from 32: by 4e-13
    acts = torch.einsum("th,eih->tei", x.double(), gu[:, I:].double()) * 32
    assert torch.equal(ref, ref.to(dtype).double()) and torch.equal(acts, acts.to(dtype).double())
    out = B.few_token_block(x.to(dtype).cuda(), router.to(dtype).cuda(), k, True, ew)
    assert torch.equal(out.double().cpu(), ref) and float(ref.abs().max()) > 0


@pytest.mark.parametrize("fmt", ["q4", "fp8"])
def test_equal_logits_go_to_the_lowest_experts(B, fmt):
    ew, vals = _random_experts(fmt, 20, 128, 128)
    x, router = _rand(4, 128, seed=1), _rand(20, 128, seed=2, scale=0.1)
    router[7:] = router[7]  # thirteen equal rows
    x[2] = 0                # a padding token: every expert ties
    out = B.few_token_block(x.cuda(), router.cuda(), 4, True, ew)
    ref = _layer(x, _route(x, router, 4, True), vals)
    assert not out[2].any()
    keep = torch.tensor([0, 1, 3])
    _check(out[keep], ref[keep], torch.bfloat16)


def test_a_mean_far_from_zero(B):
    """Tokens whose values share a large mean: the codes' offset must not swallow the digits behind it."""
    for dtype in DTYPES:
        ew, vals = _random_experts("q4", 4, 512, 256)
        x = _rand(5, 512, dtype=torch.float32, seed=3, scale=0.25).add_(4).to(dtype)
        router = _rand(4, 512, dtype=dtype, seed=5, scale=0.02)
        out = B.few_token_block(x.cuda(), router.cuda(), 2, True, ew)
        _check(out, _layer(x, _route(x, router, 2, True), vals), dtype)


@pytest.mark.parametrize("fmt", ["q4", "fp8"])
def test_a_token_that_is_not_finite_stays_alone(B, fmt):
    ew, _ = _random_experts(fmt, 6, 256, 128)
    x, router = _rand(8, 256, seed=1), _rand(6, 256, seed=2, scale=0.1)
    want = B.few_token_block(x.cuda(), router.cuda(), 2, True, ew)
    for bad in (float("nan"), float("inf")):
        y = x.clone()
        y[3, 17] = bad
        got = B.few_token_block(y.cuda(), router.cuda(), 2, True, ew)
        keep = [0, 1, 2, 4, 5, 6, 7]
        assert torch.equal(got[keep], want[keep]) and bool(torch.isnan(got[3]).all())
    r = router.clone()
    r[4, 0] = float("nan")
    assert bool(torch.isnan(B.few_token_block(x.cuda(), r.cuda(), 2, True, ew)).all())


@pytest.mark.parametrize("fmt", ["q4", "fp8"])
def test_weights_that_are_not_finite_stay_with_their_expert(B, fmt):
    E, H, I = 4, 128, 128
    ew, _ = _random_experts(fmt, E, H, I)
    x, router = torch.zeros(6, H, dtype=torch.bfloat16), torch.zeros(E, H, dtype=torch.bfloat16)
    x += _rand(6, H, seed=1) * 0.1
    x[:, :E] = 0
    for t in range(6):
        x[t, t % 3] = 8
    router[torch.arange(E), torch.arange(E)] = 8
    want = B.few_token_block(x.cuda(), router.cuda(), 1, True, ew)
    if fmt == "q4":  # expert 1's down scales: infinite
        n = ew.down.s.numel() // E
        ew.down.s[n:2 * n] = float("inf")
        ew.down._sz = ew.down._szg = None
    else:
        ew.down.q[1] = 0x7F
    got = B.few_token_block(x.cuda(), router.cuda(), 1, True, ew)
    keep = [0, 2, 3, 5]
    assert torch.equal(got[keep], want[keep]) and not bool(torch.isfinite(got[[1, 4]]).any())


def test_large_activations_do_not_overflow_the_sums(B):
    """bf16 values past fp16's range."""
    ew, vals = _random_experts("q4", 4, 256, 128)
    x, router = _rand(3, 256, seed=1, scale=3e4), _rand(4, 256, seed=2, scale=1e-6)
    out = B.few_token_block(x.cuda(), router.cuda(), 2, True, ew)
    _check(out, _layer(x, _route(x, router, 2, True), vals), torch.bfloat16)


def test_shapes_strides_and_streams(B):
    ew, _ = _random_experts("q4", 8, 256, 128)
    router = _rand(8, 256, seed=5, scale=0.1).cuda()
    base = _rand(4, 6, 264, seed=6).cuda()
    flat = base[:, :, 1:257].contiguous()
    want = B.few_token_block(flat.view(24, 256), router, 2, True, ew)
    for x in (base[:, :, 1:257], flat, flat.view(2, 2, 6, 256)):
        out = B.few_token_block(x, router, 2, True, ew)
        assert out.shape == x.shape and torch.equal(out.reshape(24, 256), want)
    assert torch.equal(B.few_token_block(flat[0, 0], router, 2, True, ew), want[0])
    odd = torch.empty(8 * 256 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(8, 256).copy_(router)
    assert torch.equal(B.few_token_block(flat, odd, 2, True, ew).reshape(24, 256), want)
    assert B.few_token_block(flat[:0], router, 2, True, ew).shape == (0, 6, 256)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    outs = []
    for i in range(9):  # calls that may overlap
        with torch.cuda.stream(streams[i % 3]):
            outs.append(B.few_token_block(flat, router, 2, True, ew))
    torch.cuda.synchronize()
    assert all(torch.equal(o.reshape(24, 256), want) for o in outs)


def test_a_token_alone_and_in_a_batch(B):
    """Which tokens share the call does not change a token's bits where the launch's split is the same."""
    ew, _ = _random_experts("fp8", 4, 256, 128)
    x, router = _rand(32, 256, seed=7).cuda(), _rand(4, 256, seed=5, scale=0.1).cuda()
    whole = B.few_token_block(x, router, 4, True, ew)
    part = B.few_token_block(x[5:25], router, 4, True, ew)
    assert torch.equal(whole[5:25], part)


def test_in_graphs(B):
    ew, _ = _random_experts("q4", 16, 256, 128)
    router, x = _rand(16, 256, seed=5, scale=0.1).cuda(), _rand(6, 256, seed=1).cuda()
    with torch.no_grad():
        B.few_token_block(x, router, 4, True, ew)
        graphs = []
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                out = B.few_token_block(x, router, 4, True, ew)
                out = B.few_token_block(out, router, 4, True, ew)  # a second layer behind the first
            graphs.append((g, out))
        for i in range(4):
            x.copy_(_rand(6, 256, seed=20 + i))
            for g, _ in graphs:
                g.replay()
            torch.cuda.synchronize()
            want = B.few_token_block(B.few_token_block(x, router, 4, True, ew), router, 4, True, ew)
            torch.cuda.synchronize()
            assert all(torch.equal(out, want) for _, out in graphs)


def test_near_the_routed_layer(B):
    """moe_block on the same experts: its 16-bit roundings apart (about ten half steps along a token's path, and the weights'
    own), the same layer.  Logits are whole numbers, so the two route alike."""
    from usaf_amd.moe import moe_block
    E, H, I, k = 16, 256, 128, 3
    ew, _ = _random_experts("q4", E, H, I)
    x, router = _rand(20, H, seed=3), torch.zeros(E, H, dtype=torch.bfloat16)
    x[:, :E] = torch.stack([torch.randperm(E, generator=torch.Generator().manual_seed(i)) for i in range(20)]).to(x.dtype) / 4
    router[torch.arange(E), torch.arange(E)] = 4
    a = B.few_token_block(x.cuda(), router.cuda(), k, True, ew).double()
    with torch.no_grad():
        b = moe_block(x.cuda(), router.cuda(), k, True, ew).double()
    rel = (a - b).norm(dim=-1) / b.norm(dim=-1)
    assert float(rel.max()) <= 10 * O.half_step(torch.bfloat16)


@pytest.mark.parametrize("fmt", ["q4", "fp8"])
def test_weights_past_32_bits(B, fmt):
    """The last of the experts, past 4 GiB of codes: as the only expert of its own, in every bit."""
    from usaf_amd.fp8 import Fp8Tensor
    from usaf_amd.moe import ExpertWeights, Q4Tensor
    E, H, I = (80 if fmt == "q4" else 40), 8192, 8192
    small, _ = _random_experts(fmt, 1, H, I)
    big = []
    for t, shape in ((small.gate_up, (E, 2 * I, H)), (small.down, (E, H, I))):
        parts = (t.q, t.s) if fmt == "fp8" else (t.q, t.s, t.z)
        wide = []
        for p in parts:
            rows = p.shape[1:] if fmt == "fp8" else p.shape
            a = torch.zeros(E * rows[0], *rows[1:], dtype=p.dtype, device="cuda")
            a[-rows[0]:] = p.reshape(rows)
            wide.append(a.view(E, *rows) if fmt == "fp8" else a)
        big.append(Fp8Tensor(*wide, shape) if fmt == "fp8" else Q4Tensor(*wide, torch.Size(shape)))
    x = _rand(2, H, seed=1).cuda()
    router = torch.zeros(E, H, dtype=torch.bfloat16, device="cuda")
    x[:, 0], router[-1, 0] = 30, 30  # both tokens to the last expert
    got = B.few_token_block(x, router, 1, True, ExpertWeights(*big))
    assert torch.equal(got, B.few_token_block(x, router[-1:], 1, True, small))


def test_patched_block_uses_it(B):
    """A patched Qwen3-MoE block with _usaf_few_tokens set takes its few-token passes here, and no others."""
    from types import SimpleNamespace
    from usaf_amd import qwen3moe_dml as Q
    E, H, I, k = 8, 256, 128, 2
    ew, _ = _random_experts("q4", E, H, I)
    router = _rand(E, H, seed=5, scale=0.1).cuda()

    class Experts(torch.nn.Module):
        forward = Q.dml_qwen3_experts_forward

    class Block(torch.nn.Module):
        forward = Q.dml_qwen3_moe_block_forward

    ex, block = Experts(), Block()
    ex._usaf_q4 = {"gate_up_proj": ew.gate_up, "down_proj": ew.down}
    block.experts, block.gate = ex, SimpleNamespace(weight=router, top_k=k, norm_topk_prob=True)
    x = _rand(2, 3, H, seed=1).cuda()
    few = B.few_token_block(x, router, k, True, ew)
    with torch.no_grad():
        routed = block(x)
        block._usaf_few_tokens = 8
        assert torch.equal(block(x), few)
        assert torch.equal(block(x.repeat(2, 1, 1)), block.__class__.forward(_without(block), x.repeat(2, 1, 1)))  # 12 tokens
    assert torch.equal(block(x.clone().requires_grad_(True)).detach(), routed)  # a gradient is wanted
    ov = ew.set_overlay("down", torch.tensor([3], device="cuda"), torch.ones(1, device="cuda"), torch.bfloat16)
    ex._usaf_q4_overlays = {"down_proj": ov}
    with torch.no_grad():
        assert not torch.equal(block(x), few)


def _without(block):
    import copy
    b = copy.copy(block)
    b.__dict__ = {k: v for k, v in block.__dict__.items() if k != "_usaf_few_tokens"}
    return b


def test_refusals(B):
    from usaf_amd.moe import ExpertWeights
    ew, _ = _random_experts("q4", 4, 128, 128)
    x, r = _rand(2, 128).cuda(), _rand(4, 128).cuda()
    call = B.few_token_block
    with pytest.raises(ValueError, match="at most 32"):
        call(_rand(33, 128).cuda(), r, 2, True, ew)
    with pytest.raises(TypeError):
        call(x, r.half(), 2, True, ew)
    with pytest.raises(TypeError):
        call(x.float(), r.float(), 2, True, ew)
    with pytest.raises(ValueError, match="fit"):
        call(x[:, :64], r, 2, True, ew)
    with pytest.raises(ValueError, match="fit"):
        call(x, r[:3], 2, True, ew)
    for k in (0, 5, -1):
        with pytest.raises(NotImplementedError):
            call(x, r, k, True, ew)
    with pytest.raises(ValueError, match="one GPU"):
        call(x.cpu(), r, 2, True, ew)
    with pytest.raises(RuntimeError, match="no backward"):
        call(x.requires_grad_(True), r, 2, True, ew)
    with torch.no_grad():
        call(x, r, 2, True, ew)
    x = x.detach()
    dense = ExpertWeights(_rand(4, 256, 128).cuda(), _rand(4, 128, 128).cuda())
    with pytest.raises(NotImplementedError):
        call(x, r, 2, True, dense)
    ew.set_overlay("down", torch.tensor([3], device="cuda"), torch.ones(1, device="cuda"), torch.bfloat16)
    with pytest.raises(NotImplementedError, match="overlays"):
        call(x, r, 2, True, ew)


@pytest.mark.parametrize("fmt", ["q4", "fp8"])
def test_under_a_trace_and_a_tangent(B, fmt):
    """A trace replays the layer, not the memory it was written to; forward-mode derivatives are refused, as on the routed path."""
    from torch.autograd import forward_ad
    ew, _ = _random_experts(fmt, 8, 256, 128)
    x, other, r = _rand(5, 256, seed=1).cuda(), _rand(5, 256, seed=2).cuda(), _rand(8, 256, seed=3, scale=0.1).cuda()
    with torch.no_grad():
        traced = torch.jit.trace(lambda v: B.few_token_block(v, r, 2, True, ew) * 2, (x,))
        for v in (other, x):
            assert torch.equal(traced(v), B.few_token_block(v, r, 2, True, ew) * 2)
    with forward_ad.dual_level():
        for args in ((forward_ad.make_dual(x, x), r), (x, forward_ad.make_dual(r, r))):
            with pytest.raises((NotImplementedError, RuntimeError), match="forward"):
                B.few_token_block(*args, 2, True, ew)


@pytest.mark.parametrize("cached", [False, True])
def test_a_streamed_models_decoding_passes(B, cached):
    """The switch on a model that the loader set up: the same bits as the layer called by itself; with trained values, and
    without the switch, the routed path; 8-bit experts attached by hand in place of the streamed ones."""
    from types import SimpleNamespace
    from torch import nn
    from usaf_amd import qwen3moe_dml as Q
    from usaf_amd.fp8 import Fp8Tensor
    from usaf_amd.moe import ExpertWeights
    from usaf_amd.moe_loader import get_quantized_cache, setup_quantized_streaming
    from usaf_amd.quantization import quantize_state_dict
    E, H, I, k = 8, 256, 128, 2

    class Experts(nn.Module):
        forward = Q.dml_qwen3_experts_forward

    class Block(nn.Module):
        forward = Q.dml_qwen3_moe_block_forward

    model, block = nn.Module(), Block()
    model.mlp, block.experts = block, Experts()
    block.gate = SimpleNamespace(weight=_rand(E, H, seed=5, scale=0.1).cuda(), top_k=k, norm_topk_prob=True)
    model.scale = nn.Parameter(torch.ones(1, dtype=torch.bfloat16), requires_grad=False)
    w = {"mlp.experts.gate_up_proj": _rand(E, 2 * I, H, dtype=torch.float16, seed=1, scale=0.05),
         "mlp.experts.down_proj": _rand(E, H, I, dtype=torch.float16, seed=2, scale=0.05)}
    kw = {"expert_cache_bytes": E * 3 * H * I * 2} if cached else {}
    setup_quantized_streaming(model, quantize_state_dict(w, device="cuda"), torch.device("cuda", 0), verbose=False,
                              expert_pattern="mlp.experts", **kw)
    cache = get_quantized_cache(model)
    q4 = cache.get_q4("mlp.experts")
    x, longer = _rand(2, 3, H, seed=3).cuda(), _rand(3, 3, H, seed=4).cuda()
    with torch.no_grad():
        want = B.few_token_block(x, block.gate.weight, k, True, ExpertWeights(q4["gate_up_proj"], q4["down_proj"]))
        routed, routed_longer = block(x), block(longer)
        assert not torch.equal(routed, want)
        block._usaf_few_tokens = 8
        for _ in range(2):
            assert torch.equal(block(x), want) and torch.equal(block(longer), routed_longer)
        eight = {n.rsplit(".", 1)[1]: Fp8Tensor.quantize(t.cuda()) for n, t in w.items()}
        block.experts._usaf_q4 = eight
        ew = ExpertWeights(eight["gate_up_proj"], eight["down_proj"])
        for _ in range(2):
            assert torch.equal(block(x), B.few_token_block(x, block.gate.weight, k, True, ew))
            assert not torch.equal(block(longer), routed_longer)
        block.experts._usaf_q4 = None
        assert torch.equal(block(x), want)
        name, at = "mlp.experts.down_proj", torch.tensor([3, 500], device="cuda")
        cache.overlays[name] = (at, torch.full((2,), 4.0, device="cuda"))
        trained = block(x)
        assert not torch.equal(trained, want)
        del block._usaf_few_tokens
        assert torch.equal(block(x), trained)
