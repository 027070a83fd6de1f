"""The routed expert layer in the forms it is served in, as cases that can be timed and compared.

Two operators of the layer and the product below the second:

* ``few``: a whole MoE layer (router, top-k, experts, weighted sum) for 1 to 32 tokens, on 4-bit or 8-bit experts
  (``usaf_amd.few.few_token_block``);
* ``linear``: the product with an 8-bit block-scaled weight, and its grad-input (``usaf_amd.fp8.fp8_linear``);
* ``experts``: the routed experts on 8-bit weights, forward and grad-input (``usaf_amd.moe.routed_experts``).

Shapes are those of the benchmark (Qwen3-30B-A3B and Mixtral-8x7B layers), of the OLMoE-1B-7B layer in the tests, one
small generic layer, and generic sizes for the product.  ``own`` chooses between the framework's calls and the plain form
in torch.  Definitions, with dt the dtype of the activations (bf16 or fp16):

* An 8-bit block of 128 values has one power-of-two scale 2^e, e the smallest integer that brings its largest magnitude to
  448 or below; its codes are e4m3, rounded to nearest even.  Activations: blocks of 1 x 128, quantized in the call;
  weights: 128 x 128, held as codes and exponents.
* A 4-bit weight is code * scale + zero of its group of 128 along the row, as a real number.
* Activations between two products are of dtype dt.  ``experts`` rounds what each of its steps gives to dt (the layer's
  convention: gate and up, the gated activation, each expert's output, each gradient); ``few`` rounds the gated
  activation, the operand of the second product, and the output.
"""
from __future__ import annotations

import torch

own = False

SHAPES = {  # experts, hidden, intermediate, experts per token
    "qwen3": (128, 2048, 768, 8),
    "mixtral": (8, 4096, 14336, 2),
    "olmoe": (64, 2048, 1024, 8),
    "small": (32, 1024, 512, 4),
    "odd": (13, 640, 384, 3),
}
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
BLOCK = 128


def listed():
    return [
        # one decoded token through a 4-bit layer: latency and launches
        {"name": "few_1_q4", "kind": "few", "shape": "qwen3", "T": 1, "format": "q4", "dtype": "bf16", "norm": True},
        # a decode step of a batch of 24 sequences: about 100 of 128 experts are read
        {"name": "few_24_q4", "kind": "few", "shape": "qwen3", "T": 24, "format": "q4", "dtype": "bf16", "norm": True},
        # a few tokens on large experts: all of the layer's weights are read
        {"name": "few_7_q4_mixtral", "kind": "few", "shape": "mixtral", "T": 7, "format": "q4", "dtype": "fp16", "norm": True},
        # 8-bit experts: two tokens (a short draft that is verified), and a full batch
        {"name": "few_2_fp8", "kind": "few", "shape": "qwen3", "T": 2, "format": "fp8", "dtype": "bf16", "norm": True},
        {"name": "few_32_fp8", "kind": "few", "shape": "olmoe", "T": 32, "format": "fp8", "dtype": "bf16", "norm": False},
        # one token through a projection: the weight is read once
        {"name": "linear_1", "kind": "linear", "M": 1, "N": 4096, "K": 2048, "dtype": "bf16", "grad": False},
        # a ragged batch, sizes that fill no tile, forward and grad-input
        {"name": "linear_odd", "kind": "linear", "M": 333, "N": 1411, "K": 2027, "dtype": "fp16", "grad": True},
        # a frozen projection in training, forward and grad-input
        {"name": "linear_4096", "kind": "linear", "M": 4096, "N": 4096, "K": 2048, "dtype": "bf16", "grad": True},
        # the largest: a prefill of 8,192 tokens through a wide projection
        {"name": "linear_8192", "kind": "linear", "M": 8192, "N": 14336, "K": 4096, "dtype": "bf16", "grad": False},
        # a training microbatch on frozen experts: 16 rows for each expert on average
        {"name": "experts_256", "kind": "experts", "shape": "qwen3", "T": 256, "dtype": "bf16", "skew": 0.0, "grad": True},
        # a prefill with a skewed routing
        {"name": "experts_2048", "kind": "experts", "shape": "olmoe", "T": 2048, "dtype": "fp16", "skew": 1.1, "grad": False},
        # a training step of 4,096 tokens on frozen experts
        {"name": "experts_4096", "kind": "experts", "shape": "qwen3", "T": 4096, "dtype": "bf16", "skew": 0.0, "grad": True},
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(low * (high / low) ** rng.random()))))


def draw(rng):
    dtype = rng.choice(["bf16", "fp16"])
    kind = rng.choice(["few", "few", "linear", "linear", "experts"])
    if kind == "few":
        return {"kind": "few", "shape": rng.choice(list(SHAPES)), "T": _log_int(rng, 1, 32), "format": rng.choice(["q4", "fp8"]),
                "dtype": dtype, "norm": rng.random() < 0.5}
    if kind == "linear":
        M, N, K = _log_int(rng, 1, 8192), _log_int(rng, 64, 14336), _log_int(rng, 64, 4096)
        return {"kind": "linear", "M": M, "N": N, "K": K, "dtype": dtype,
                "grad": rng.random() < 0.5 and 2 * M * N * K <= 8192 * 14336 * 4096}
    shape = rng.choice(["qwen3", "olmoe", "small", "odd"])
    return {"kind": "experts", "shape": shape, "T": _log_int(rng, 8, 4096), "dtype": dtype, "skew": rng.choice([0.0, 1.1]),
            "grad": rng.random() < 0.5}


# ---------------------------------------------------------------------------
# what a program holds before the call
# ---------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _weight8(gen, *shape):
    """Codes (e4m3 bits, columns padded with zeros to whole blocks) and E8M0 exponents (e + 127) of a weight of about 0.02."""
    *lead, rows, cols = shape
    wide = -(-cols // BLOCK) * BLOCK
    q = torch.zeros(*lead, rows, wide, dtype=torch.uint8, device="cuda")
    flat, at = q.view(-1, wide), 0
    while at < flat.shape[0]:  # in pieces: the largest weight's normal numbers in 32 bits would take 6 GB
        part = flat[at:at + (1 << 26) // wide + 1]
        v = (torch.randn(part.shape[0], cols, device="cuda", generator=gen) * 96).clamp_(-448, 448)
        part[:, :cols] = v.to(torch.float8_e4m3fn).view(torch.uint8)
        at += part.shape[0]
    e = torch.randint(127 - 13, 127 - 11, (*lead, -(-rows // BLOCK), wide // BLOCK), device="cuda", generator=gen)
    return q, e.to(torch.uint8)


def _weight4(gen, *shape):
    """4-bit codes, two a byte, low nibble first, with fp16 scale and zero for each 128 of a row: values of about 0.02."""
    n = 1
    for d in shape:
        n *= d
    q = torch.randint(0, 256, (n // BLOCK, BLOCK // 2), dtype=torch.uint8, device="cuda", generator=gen).view(torch.int8)
    s = (0.0035 + 0.002 * torch.rand(n // BLOCK, device="cuda", generator=gen)).half()
    return q, s, (-7.5 * s.float() * (0.9 + 0.2 * torch.rand(n // BLOCK, device="cuda", generator=gen))).half()


def prepare(case, seed):
    gen, dt = _gen(seed), DTYPES[case["dtype"]]
    st = {"case": dict(case)}
    if case["kind"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        st["w"] = _weight8(gen, N, K)
        st["x"] = torch.randn(M, K, device="cuda", generator=gen).to(dt).requires_grad_(case["grad"])
        if case["grad"]:
            st["dy"] = torch.randn(M, N, device="cuda", generator=gen).to(dt)
        if own:
            from usaf_amd.fp8 import Fp8Tensor
            st["layer"] = Fp8Tensor(*st["w"], (N, K))
        return st
    E, H, I, k = SHAPES[case["shape"]]
    T, four = case["T"], case.get("format") == "q4"
    make = _weight4 if four else _weight8
    st["gate_up"], st["down"] = make(gen, E, 2 * I, H), make(gen, E, H, I)
    st["x"] = torch.randn(T, H, device="cuda", generator=gen).to(dt)
    if case["kind"] == "few":
        st["router"] = (torch.randn(E, H, device="cuda", generator=gen) * (1.5 / H ** 0.5)).to(dt)
    else:
        # a routing as the router leaves it: k experts a token, the popular ones first under a skew
        pop = -case["skew"] * torch.log(torch.arange(1, E + 1, device="cuda", dtype=torch.float32))
        p = torch.softmax(torch.randn(T, E, device="cuda", generator=gen) + pop, dim=-1)
        top = p.topk(k, dim=-1)
        w = torch.zeros_like(p).scatter_(1, top.indices, top.values / top.values.sum(-1, keepdim=True))
        st["weights"] = w.to(dt).requires_grad_(case["grad"])
        st["x"].requires_grad_(case["grad"])
        if case["grad"]:
            st["dy"] = torch.randn(T, H, device="cuda", generator=gen).to(dt)
    if own:
        from usaf_amd.moe import ExpertWeights, Q4Tensor
        if four:
            wrap = lambda q, shape: Q4Tensor(*q, torch.Size(shape))  # noqa: E731
        else:
            from usaf_amd.fp8 import Fp8Tensor
            wrap = lambda q, shape: Fp8Tensor(*q, shape)  # noqa: E731
        st["layer"] = ExpertWeights(wrap(st["gate_up"], (E, 2 * I, H)), wrap(st["down"], (E, H, I)))
    return st


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(st):
    case = st["case"]
    if case["kind"] == "few":
        k = SHAPES[case["shape"]][3]
        if own:
            from usaf_amd.few import few_token_block
            with torch.no_grad():
                return {"out": few_token_block(st["x"], st["router"], k, case["norm"], st["layer"])}
        return {"out": _plain_few(st, k)}
    if not own:
        return _plain_linear(st) if case["kind"] == "linear" else _plain_experts(st)
    x, w = st["x"], st.get("weights")
    if case["kind"] == "linear":
        from usaf_amd.fp8 import fp8_linear as call
        args = (x, st["layer"])
    else:
        from usaf_amd.moe import routed_experts as call
        args = (x, w, st["layer"])
    if not case["grad"]:
        with torch.no_grad():
            return {"out": call(*args)}
    x.grad = None
    if w is not None:
        w.grad = None
    out = call(*args)
    out.backward(st["dy"])
    return {"out": out.detach(), "dx": x.grad, **({} if w is None else {"dw": w.grad})}


# ---------------------------------------------------------------------------
# the plain form: elementary operations in 32 bits
# ---------------------------------------------------------------------------

def _values8(weight, cols):
    """The fp32 values of a block-scaled weight."""
    q, e = weight
    rows, wide = q.shape[-2:]
    scale = torch.exp2(e.float() - 127).repeat_interleave(BLOCK, -2)[..., :rows, :]
    v = q.view(torch.float8_e4m3fn).float().view(*q.shape[:-1], wide // BLOCK, BLOCK) * scale.unsqueeze(-1)
    return v.view(*q.shape[:-1], wide)[..., :cols]


def _values4(weight, shape):
    q, s, z = weight
    b = q.view(torch.uint8)
    codes = torch.stack([b & 15, b >> 4], dim=-1).view(-1, BLOCK).float()
    return (codes * s.float()[:, None] + z.float()[:, None]).view(shape)


def _quantized(x):
    """fp32 values of the rows of x after the 8-bit quantization in blocks of 128 along the row."""
    rows, cols = x.shape
    v = torch.nn.functional.pad(x.float(), (0, -cols % BLOCK)).view(rows, -1, BLOCK)
    m, e = torch.frexp(v.abs().amax(-1, keepdim=True))  # largest = m 2^e, m in [1/2, 1); 448 = 7/8 2^9
    scale = torch.exp2((torch.where(m > 0.875, e - 8, e - 9)).clamp_(-120, 120).float())
    return ((v / scale).to(torch.float8_e4m3fn).float() * scale).view(rows, -1)[:, :cols]


@torch.no_grad()
def _plain_linear(st):
    dt = st["x"].dtype
    w = _values8(st["w"], st["case"]["K"])
    out = {"out": (_quantized(st["x"]) @ w.t()).to(dt)}
    if st["case"]["grad"]:
        out["dx"] = (_quantized(st["dy"]) @ w).to(dt)
    return out


def _round(v, dt):
    return v.to(dt).float()


@torch.no_grad()
def _plain_experts(st):
    E, H, I, _ = SHAPES[st["case"]["shape"]]
    dt, x, w = st["x"].dtype, st["x"].detach(), st["weights"].detach().float()
    wgu, wd = _values8(st["gate_up"], H), _values8(st["down"], I)
    # the routed pairs by expert, each expert's tokens at the rows of a batch as long as the longest expert's
    expert, token = (w.t() != 0).nonzero(as_tuple=True)
    counts = torch.bincount(expert, minlength=E)
    place = torch.arange(expert.numel(), device="cuda") - (counts.cumsum(0) - counts)[expert]
    longest = int(counts.max())

    def batch(rows):  # [pairs, C] -> [E, longest, C]
        b = torch.zeros(E, longest, rows.shape[1], device="cuda")
        b[expert, place] = rows
        return b

    def tokens(pairs):  # the sum over each token's pairs
        return torch.zeros(x.shape[0], H, device="cuda").index_add_(0, token, pairs)

    pw = w[token, expert][:, None]
    gu = _round(torch.bmm(batch(_quantized(x)[token]), wgu.transpose(1, 2))[expert, place], dt)
    gate, up = gu[:, :I], gu[:, I:]
    sig = torch.sigmoid(gate)
    act = _round(_round(gate * sig, dt) * up, dt)
    y = _round(torch.bmm(batch(_quantized(act)), wd.transpose(1, 2))[expert, place], dt)
    out = {"out": tokens(pw * y).to(dt)}
    if st["case"]["grad"]:
        dout = st["dy"].float()[token]
        out["dw"] = torch.zeros_like(w).index_put_((token, expert), (dout * y).sum(1)).to(dt)
        dact = _round(torch.bmm(batch(_quantized(_round(pw * dout, dt))), wd)[expert, place], dt)
        dsilu = _round(dact * up, dt)
        dgate = _round(dsilu * sig * (1 + gate * (1 - sig)), dt)
        dup = _round(dact * _round(gate * sig, dt), dt)
        dxs = _round(torch.bmm(batch(_quantized(torch.cat([dgate, dup], 1))), wgu)[expert, place], dt)
        out["dx"] = tokens(dxs).to(dt)
    return out


@torch.no_grad()
def _plain_few(st, k):
    E, H, I, _ = SHAPES[st["case"]["shape"]]
    T, dt, x = st["case"]["T"], st["x"].dtype, st["x"].float()
    # in 64 bits: which experts are chosen hangs on differences far below the products' own size
    p = torch.softmax(st["x"].double() @ st["router"].double().t(), dim=-1)
    top, choice = torch.sort(p, dim=-1, descending=True, stable=True)
    top, choice = top[:, :k].float(), choice[:, :k]
    if st["case"]["norm"]:
        top = top / top.sum(-1, keepdim=True)
    # each pair with its expert's weights, or where the pairs are more than the experts, every expert with every token
    if T * k < E:
        pick = choice.reshape(-1)
        rows = x.repeat_interleave(k, 0)[:, None, :]
    else:
        pick = torch.arange(E, device="cuda")
        rows = x.expand(E, T, H)
    if st["case"]["format"] == "q4":
        take = lambda w, r, c: _values4([t.view(E, -1, *t.shape[1:])[pick].flatten(0, 1) for t in w], (-1, r, c))  # noqa: E731
    else:
        take = lambda w, r, c: _values8([t[pick] for t in w], c)  # noqa: E731
    gate, up = torch.bmm(rows, take(st["gate_up"], 2 * I, H).transpose(1, 2)).split(I, dim=-1)
    act = _round(gate * torch.sigmoid(gate) * up, dt)
    y = torch.bmm(act, take(st["down"], H, I).transpose(1, 2))
    if T * k < E:
        return (y.view(T, k, H) * top[:, :, None]).sum(1).to(dt)
    w = torch.zeros(T, E, device="cuda").scatter_(1, choice, top)
    return (y * w.t()[:, :, None]).sum(0).to(dt)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    if case["kind"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        passes = 2 if case["grad"] else 1
        blocks = -(-N // BLOCK) * -(-K // BLOCK)
        return {"bytes": passes * (2 * M * (N + K) + N * K + blocks), "flops": passes * 2 * M * N * K}
    E, H, I, k = SHAPES[case["shape"]]
    T = case["T"]
    used = E * (1 - (1 - k / E) ** T)  # experts some token selects
    weights = used * 3 * H * I * (0.53125 if case.get("format") == "q4" else 1)
    flops = 2 * T * k * 3 * H * I
    if case["kind"] == "few":
        return {"bytes": weights + 2 * E * H + 4 * T * H, "flops": flops + 2 * T * E * H}
    if case["grad"]:
        return {"bytes": 2 * weights + 10 * T * H + 8 * T * E, "flops": 2 * flops}
    return {"bytes": weights + 4 * T * H + 4 * T * E, "flops": flops}


# ---------------------------------------------------------------------------
# the same outputs in 64 bits
# ---------------------------------------------------------------------------

def _e4m3(v):
    """Nearest e4m3 number, ties to even, of float64 values up to 448."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3)  # 3 bits behind the first; 2^-9 at the low end
    return torch.round(v / step) * step


def _q64(x):
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for a in range(0, x.shape[1], BLOCK):
        v = x[:, a:a + BLOCK].double()
        largest = v.abs().amax(1, keepdim=True).clamp_min(2.0 ** -120)
        scale = torch.exp2(torch.ceil(torch.log2(largest / 448)))
        scale = torch.where(largest / scale > 448, scale * 2, torch.where(largest * 2 / scale <= 448, scale / 2, scale))
        out[:, a:a + BLOCK] = _e4m3(v / scale) * scale
    return out


def _w64(weight, rows, cols, e=None):
    """A weight, or its matrix e, in 64 bits: (codes, E8M0 exponents) of the 8-bit format, (codes, scale, zero) of the 4-bit one."""
    if len(weight) == 3:
        groups = rows * (cols // BLOCK)
        q, s, z = (t[e * groups:(e + 1) * groups] for t in weight)
        b = q.view(torch.uint8).long()
        codes = torch.empty(groups, BLOCK, dtype=torch.float64, device=q.device)
        codes[:, 0::2], codes[:, 1::2] = (b % 16).double(), torch.div(b, 16, rounding_mode="floor").double()
        return (codes * s.double()[:, None] + z.double()[:, None]).reshape(rows, cols)
    q, x = weight if e is None else (weight[0][e], weight[1][e])
    out = torch.empty(rows, cols, dtype=torch.float64, device=q.device)
    block_of_row = torch.arange(rows, device=q.device) // BLOCK
    for a in range(x.shape[1]):
        part = q[:, a * BLOCK:min(cols, (a + 1) * BLOCK)].contiguous().view(torch.float8_e4m3fn).double()
        out[:, a * BLOCK:a * BLOCK + part.shape[1]] = part * torch.pow(2.0, x[block_of_row, a].double() - 127)[:, None]
    return out


@torch.no_grad()
def exact(case, seed):
    st = prepare(case, seed)
    dt, x = DTYPES[case["dtype"]], st["x"].detach()
    if case["kind"] == "linear":
        w = _w64(st["w"], case["N"], case["K"])
        out = {"out": _q64(x) @ w.t()}
        if case["grad"]:
            out["dx"] = _q64(st["dy"]) @ w
        return out
    E, H, I, k = SHAPES[case["shape"]]
    few = case["kind"] == "few"
    if few:
        p = torch.exp(x.double() @ st["router"].double().t())
        p = p / p.sum(1, keepdim=True)
        order = torch.argsort(-p, dim=1, stable=True)
        chosen = torch.zeros_like(p).scatter_(1, order[:, :k], 1.0)
        w = p * chosen
        if case["norm"]:
            w = w / w.sum(1, keepdim=True)
    else:
        w = st["weights"].detach().double()
    r = (lambda v: v) if few else (lambda v: v.to(dt).double())
    x8 = x.double() if few else _q64(x)
    out = torch.zeros(x.shape, dtype=torch.float64, device="cuda")
    grad = case.get("grad", False)
    if grad:
        dout, dx, dw = st["dy"].double(), torch.zeros_like(out), torch.zeros_like(w)
    for e in range(E):
        rows = w[:, e].nonzero().reshape(-1)
        if not rows.numel():
            continue
        wgu, wd = _w64(st["gate_up"], 2 * I, H, e), _w64(st["down"], H, I, e)
        gu = r(x8[rows] @ wgu.t())
        gate, up = gu[:, :I], gu[:, I:]
        sig = 1 / (1 + torch.exp(-gate))
        act = (r(gate * sig) * up).to(dt)
        we = w[rows, e:e + 1]
        y = r((act.double() if few else _q64(act)) @ wd.t())
        out[rows] += we * y
        if grad:
            de = dout[rows]
            dw[rows, e] = (de * y).sum(1)
            da = r(_q64((we * de).to(dt)) @ wd)
            dgate = r(r(da * up) * sig * (1 + gate * (1 - sig)))
            dup = r(da * r(gate * sig))
            dx[rows] += r(_q64(torch.cat([dgate, dup], 1).to(dt)) @ wgu)
    return {"out": out, "dx": dx, "dw": dw} if grad else {"out": out}
