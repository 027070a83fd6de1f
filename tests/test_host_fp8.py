"""Argument checks of the 8-bit block format: no GPU work."""
import ctypes

import pytest
import torch

from usaf_amd import _native as N
from usaf_amd import fp8
from usaf_amd.few import few_token_block
from usaf_amd.moe import ExpertWeights, Q4Tensor, routed_experts


def _t(*shape):
    *lead, r, c = shape
    return fp8.Fp8Tensor(torch.zeros(*lead, r, -(-c // 128) * 128, dtype=torch.uint8),
                         torch.zeros(*lead, -(-r // 128), -(-c // 128), dtype=torch.uint8), shape)


def test_tensor_shapes():
    assert _t(5, 130).numel() == 650 and _t(2, 5, 130).nbytes() == 2 * (5 * 256 + 2)
    q, s = torch.zeros(5, 256, dtype=torch.uint8), torch.zeros(1, 2, dtype=torch.uint8)
    for bad in [(5, 129, 1), (5,), (0, 130), (5, 300), (6, 130)]:
        with pytest.raises(ValueError):
            fp8.Fp8Tensor(q, s, bad)
    with pytest.raises(TypeError):
        fp8.Fp8Tensor(q.float(), s, (5, 130))
    with pytest.raises(ValueError):
        fp8.Fp8Tensor(q.t().contiguous().t(), s, (5, 130))
    with pytest.raises(ValueError):
        fp8.Fp8Tensor(torch.zeros(5 * 256 + 1, dtype=torch.uint8)[1:].view(5, 256), s, (5, 130))
    assert fp8.Fp8Tensor(q.view(torch.float8_e4m3fn), s, (5, 130)).q.dtype == torch.uint8


def test_linear_refuses():
    w = _t(64, 128)
    x = torch.zeros(3, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU"):
        fp8.fp8_linear(x, w)
    with pytest.raises(ValueError, match="fit"):
        fp8.fp8_linear(x[:, :100], w)
    with pytest.raises(ValueError):
        fp8.fp8_linear(x, _t(2, 64, 128))
    with pytest.raises(TypeError):
        fp8.fp8_linear(x.float(), w)
    with pytest.raises(ValueError):
        fp8.Fp8Tensor.quantize(torch.zeros(3))
    with pytest.raises(ValueError):
        fp8.Fp8Tensor.quantize(torch.zeros(0, 3))


def test_expert_weights_refuse():
    ExpertWeights(_t(3, 256, 256), _t(3, 256, 128))
    with pytest.raises(NotImplementedError):
        ExpertWeights(_t(3, 192, 256), _t(3, 256, 96))
    with pytest.raises(TypeError):
        ExpertWeights(torch.zeros(3, 256, 256), _t(3, 256, 128))
    with pytest.raises(ValueError):
        ExpertWeights(_t(3, 256, 256), _t(3, 128, 256))


def test_entry_points_check_their_arguments():
    lib, p, odd = N.load(), ctypes.c_void_p(4096), ctypes.c_void_p(4097)
    inval, ok = N.USAF_ERR_INVALID, N.USAF_OK
    rows = lib.usaf_hip_fp8_quantize_rows
    assert rows(None, N.BF16, 0, 8, 8, None, None, None, None) == ok
    assert rows(None, N.BF16, 1, 8, 8, None, p, p, None) == inval
    assert rows(p, N.BF16, 1, 8, 7, None, p, p, None) == inval
    assert rows(p, N.F32, 1, 8, 8, None, p, p, None) == inval
    assert rows(p, N.BF16, 1, 8, 8, None, odd, p, None) == inval
    assert rows(p, N.BF16, -1, 8, 8, None, p, p, None) == inval
    assert rows(p, N.BF16, 1 << 62, 8, 8, None, p, p, None) == inval
    gemm = lib.usaf_hip_fp8_gemm
    assert gemm(None, None, 0, None, 0, None, None, None, 1, 8, 8, N.BF16, 0, None, None) == ok
    assert gemm(p, p, 1, None, 1, p, p, None, 2, 8, 8, N.BF16, 0, p, None) == inval
    assert gemm(p, p, 1, None, 1, p, p, None, 1, 8, 0, N.BF16, 0, p, None) == inval
    assert gemm(p, p, 1, None, 1, p, p, None, 1, 8, 8, N.F32, 0, p, None) == inval
    assert gemm(odd, p, 1, None, 1, p, p, None, 1, 8, 8, N.BF16, 0, p, None) == inval
    assert gemm(p, odd, 1, None, 1, p, p, None, 1, 8, 8, N.BF16, 0, p, None) == inval
    assert gemm(p, p, 1, None, 1, p, p, None, 1, 8, 8, N.BF16, 0, odd, None) == inval
    assert gemm(p, p, 1, None, 2, p, p, None, 1, 8, 8, N.BF16, 0, p, None) == inval
    assert gemm(p, p, 1 << 33, p, 1, p, p, None, 1, 8, 8, N.BF16, 0, p, None) == N.USAF_ERR_UNSUPPORTED
    assert gemm(p, p, 1 << 40, None, 1 << 40, p, p, None, 1, 8, 8, N.BF16, 0, p, None) == inval
    assert gemm(p, p, 1, None, 1, p, p, p, 256, 8, 8, N.BF16, 0, p, None) == N.USAF_ERR_UNSUPPORTED
    up, up_ok = lib.usaf_hip_fp8_gate_up, lib.usaf_hip_fp8_gate_up_ok
    assert up(None, None, 0, None, 0, None, None, None, 1, 128, 8, N.BF16, None, None, None) == ok
    assert up(p, p, 1, None, 1, p, p, p, 1, 100, 8, N.BF16, p, p, None) == inval
    assert up(p, p, 1, None, 1, p, p, None, 1, 128, 8, N.BF16, p, p, None) == inval
    assert up(p, p, 1, None, 1, p, p, p, 1, 128, 8, N.F32, p, p, None) == inval
    assert up(p, p, 1, None, 1, p, p, p, 1, 128, 0, N.BF16, p, p, None) == inval
    for bad in [dict(q=None), dict(q=odd), dict(s=None), dict(w=odd), dict(a=None)]:
        v = {**dict(a=p, w=p, q=p, s=p), **bad}
        assert up(v["a"], p, 1, None, 1, v["w"], p, p, 1, 128, 8, N.BF16, v["q"], v["s"], None) == inval, bad
    assert [up_ok(*a) for a in [(4, 4, 128, 256), (0, 4, 128, 256), (16384, 64, 1024, 2048), (16384, 256, 1024, 2048)]] == [0, 0, 1, 0]
    assert up(p, p, 4, None, 4, p, p, p, 4, 128, 256, N.BF16, p, p, None) == N.USAF_ERR_UNSUPPORTED
    fwd, bwd = lib.usaf_hip_fp8_experts_fwd, lib.usaf_hip_fp8_experts_bwd
    fw, bw = lib.usaf_hip_fp8_experts_fwd_ws_bytes, lib.usaf_hip_fp8_experts_bwd_ws_bytes
    assert [fw(3, 128), fw(0, 128), fw(-1, 128), bw(3, 256, 128), bw(-1, 8, 8)] == [3 * 132, 0, -1, 1024 + 3 * 256, -1]
    good = dict(x=p, xs=p, T=3, tok=p, offs=p, S=3, E=2, H=256, I=128, dt=N.BF16, gu=p, gus=p, dn=p, dns=p, keep=p, act=p, y=p,
                ws=p, ws_bytes=3 * 132, stream=None)
    assert fwd(*{**good, "S": 0, "ws": None, "ws_bytes": 0}.values()) == ok
    for bad in [dict(H=100), dict(I=100), dict(tok=None), dict(offs=None), dict(y=None), dict(ws=None), dict(ws=odd),
                dict(ws_bytes=3 * 132 - 1), dict(x=None), dict(keep=None), dict(dt=N.F32), dict(x=odd), dict(S=-1)]:
        assert fwd(*{**good, **bad}.values()) == inval, bad
    assert fwd(*{**good, "keep": None, "act": None}.values()) == N.USAF_ERR_UNSUPPORTED  # few slots keep gu
    good = dict(dout=p, y=p, gu=p, tok=p, w=p, offs=p, S=3, E=2, H=256, I=128, dt=N.BF16, dn=p, dns=p, gut=p, guts=p, dcur=None,
                dgu=None, dx=p, dw=p, ws=p, ws_bytes=1024 + 768, stream=None)
    assert bwd(*{**good, "S": 0, "ws": None, "ws_bytes": 0}.values()) == ok
    for bad in [dict(H=100), dict(I=100), dict(gu=None), dict(dx=None), dict(ws=None), dict(ws=odd), dict(ws_bytes=1024 + 767),
                dict(dout=None), dict(dout=odd), dict(w=None), dict(dw=None), dict(dcur=odd), dict(dt=N.F32), dict(E=0)]:
        assert bwd(*{**good, **bad}.values()) == inval, bad
    linear = lib.usaf_hip_fp8_linear
    assert [lib.usaf_hip_fp8_linear_ws_bytes(m, k) for m, k in ((40, 130), (3, 130), (0, 5), (-1, 5))] == [40 * (256 + 4), 0, 0, -1]
    assert linear(None, N.BF16, 0, 8, 8, None, None, 8, None, None, 0, None) == ok
    assert linear(p, N.BF16, 40, 8, 8, p, p, 8, p, p, 40 * 132 - 1, None) == inval
    assert linear(p, N.BF16, 40, 8, 8, p, p, 8, p, None, 1 << 20, None) == inval
    for m in (1, 40):
        assert linear(p, N.BF16, m, 8, 7, p, p, 8, p, p, 1 << 20, None) == inval
        assert linear(p, N.F32, m, 8, 8, p, p, 8, p, p, 1 << 20, None) == inval
        assert linear(p, N.BF16, m, 8, 8, odd, p, 8, p, p, 1 << 20, None) == inval
        assert linear(p, N.BF16, m, 8, 8, p, p, -8, p, p, 1 << 20, None) == inval
        assert linear(None, N.BF16, m, 8, 8, p, p, 8, p, p, 1 << 20, None) == inval
        assert linear(p, N.BF16, m, 8, 8, p, None, 8, p, p, 1 << 20, None) == inval
        assert linear(p, N.BF16, m, 8, 8, p, p, 8, None, p, 1 << 20, None) == inval
    assert lib.usaf_hip_fp8_swiglu(p, 1, 100, N.BF16, p, p, p, p, None) == inval
    assert lib.usaf_hip_fp8_swiglu(p, 1, 128, N.BF16, None, p, p, p, None) == inval
    assert lib.usaf_hip_fp8_swiglu(None, 0, 128, N.BF16, None, None, None, None, None) == ok
    assert lib.usaf_hip_fp8_swiglu_bwd(p, odd, 1, 128, N.BF16, p, p, p, p, None) == inval
    assert lib.usaf_hip_fp8_quantize_weight(p, N.F32, 1, 1 << 25, 8, p, p, None) == inval
    assert lib.usaf_hip_fp8_quantize_weight(p, 7, 1, 8, 8, p, p, None) == inval
    assert lib.usaf_hip_fp8_dequantize(None, p, 1, 8, 8, p, N.F32, None) == inval
    assert lib.usaf_hip_fp8_transpose(odd, p, 1, 8, 8, p, p, None) == inval
    assert [lib.usaf_hip_fp8_scale_stride(c) for c in (0, 1, 512, 513, -1)] == [0, 4, 4, 8, -1]
    few, need = lib.usaf_hip_moe_few, lib.usaf_hip_moe_few_ws_bytes
    size = need(2, 4, 2, 128, 128)
    assert size > 0 and need(0, 4, 2, 128, 128) == 0 and need(32, 256, 16, 16384, 65536) < 2 << 30
    assert all(need(*a) == -1 for a in [(33, 4, 2, 128, 128), (-1, 4, 2, 128, 128), (2, 257, 2, 128, 128), (2, 4, 5, 128, 128),
                                        (2, 4, 0, 128, 128), (2, 32, 17, 128, 128), (2, 4, 2, 100, 128), (2, 4, 2, 128, 100),
                                        (2, 4, 2, 16512, 128), (2, 4, 2, 128, 65664), (2, 4, 2, 0, 128), (2, 0, 0, 128, 128)])
    good = dict(x=p, T=2, H=128, router=p, E=4, k=2, norm=1, dt=N.BF16, I=128, eight=1, gu=p, gs=p, dn=p, ds=p, out=p, ws=p,
                ws_bytes=size, stream=None)
    assert few(*{**good, "T": 0, "x": None, "ws": None, "ws_bytes": 0}.values()) == ok
    for bad in [{"x": None}, {"router": None}, {"gu": None}, {"gs": None}, {"dn": None}, {"ds": None}, {"out": None}, {"ws": None},
                {"x": odd}, {"router": odd}, {"gu": odd}, {"dn": odd}, {"ws": odd}, {"out": odd}, {"ws_bytes": 64}, {"dt": N.F32},
                {"eight": 0, "gs": odd}, {"eight": 0, "ds": odd}]:
        assert few(*{**good, **bad}.values()) == inval, bad
    for bad in [{"T": 33}, {"H": 130}, {"I": 64}, {"E": 300}, {"k": 5}]:
        assert few(*{**good, **bad}.values()) != ok, bad


def test_capture_refuses_what_is_kept_or_wants_a_gradient(monkeypatch):
    """A tensor first built in a capture would hold nothing until the replay; captured training steps are switched off."""
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    w = _t(128, 128)
    with pytest.raises(RuntimeError, match="captured"):
        w.transposed()
    assert w._t is None
    q4 = Q4Tensor(torch.zeros(512, 64, dtype=torch.int8), torch.ones(512, dtype=torch.float16),
                  torch.zeros(512, dtype=torch.float16), torch.Size((2, 256, 128)))
    with pytest.raises(RuntimeError, match="captured"):
        q4.scale_zero_by_group()
    assert q4._szg is None
    x = torch.zeros(3, 128, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="captured"):
        routed_experts(x, torch.zeros(3, 2, dtype=torch.bfloat16), ExpertWeights(_t(2, 256, 128), _t(2, 128, 128)))


def test_backward_is_not_captured(monkeypatch):
    """Of a forward pass before the capture: as the forward pass with a gradient."""
    from types import SimpleNamespace
    from usaf_amd import moe
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    dy = torch.zeros(3, 128, dtype=torch.bfloat16)
    w = _t(128, 128)
    w._t = _t(128, 128)  # built before
    with torch.no_grad():
        with pytest.raises(RuntimeError, match="captured"):
            fp8.Fp8LinearFn.backward(SimpleNamespace(w=w, dtype=dy.dtype), dy)
        ctx = SimpleNamespace(saved_tensors=(dy, None, None, dy), b=SimpleNamespace(n_slots=3), capture=None,
                              ew=ExpertWeights(_t(2, 256, 128), _t(2, 128, 128)), needs_input_grad=(True,) * 9)
        with pytest.raises(RuntimeError, match="captured"):
            moe._fp8_experts_backward(ctx, dy, torch.zeros(3, 2, dtype=torch.bfloat16))


def test_overlays_on_8_bit_experts_are_refused():
    """Trained values are held over 4-bit weights only: never left out in silence."""
    ew = ExpertWeights(_t(2, 256, 128), _t(2, 128, 128))
    ew.overlays["down"] = object()  # as a patched module's overlays are attached
    with pytest.raises(NotImplementedError, match="overlay"):
        routed_experts(torch.zeros(3, 128, dtype=torch.bfloat16), torch.zeros(3, 2, dtype=torch.bfloat16), ew)


def test_no_launch_on_cpu_tensors():
    """A CPU tensor's device has no stream: every entry point asks for one before it launches."""
    with pytest.raises(ValueError, match="GPU"):
        N.stream_ptr(torch.device("cpu"))
    x = torch.zeros(2, 128, dtype=torch.bfloat16)
    ew = ExpertWeights(_t(2, 256, 128), _t(2, 128, 128))
    for call in (lambda: fp8.quantize_rows(x), lambda: routed_experts(x, torch.ones(2, 2, dtype=torch.bfloat16), ew),
                 lambda: _t(64, 128).transposed(), lambda: _t(64, 128).dequantize(),
                 lambda: few_token_block(x, torch.zeros(2, 128, dtype=torch.bfloat16), 1, True, ew)):
        with pytest.raises((ValueError, RuntimeError, AssertionError)):
            call()


def test_followed_by_a_trace_or_a_tangent():
    """What requires_grad does not show: forward-mode derivatives and traces."""
    from torch.autograd import forward_ad
    x, seen = torch.ones(3), []

    def f(v):
        seen.append(N.followed(v))
        return v * 2

    assert not N.followed(x) and not N.followed(x.clone().requires_grad_(True))
    with torch.no_grad():
        torch.jit.trace(f, (x,), check_trace=False)
    assert seen == [True]
    with forward_ad.dual_level():
        assert not N.followed(x) and N.followed(x, forward_ad.make_dual(x, x))
        for call in (fp8.quantize_rows, fp8.Fp8Tensor.quantize):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call(forward_ad.make_dual(torch.ones(2, 128, dtype=torch.bfloat16), torch.ones(2, 128, dtype=torch.bfloat16)))
    with pytest.raises(RuntimeError, match="trace"):
        torch.jit.trace(lambda v: v + _t(2, 128).dequantize(), (x,), check_trace=False)


class _OnGpu(torch.Tensor):
    """A CPU tensor that says it is on the GPU."""
    is_cuda = True

    @classmethod
    def __torch_function__(cls, func, types, args=(), kwargs=None):
        return super().__torch_function__(func, types, args, kwargs or {})


@pytest.mark.parametrize("call", ["linear", "few"])
def test_forward_mode_derivatives_are_refused(call, monkeypatch):
    """Not left out of the output, with the launch replaced by an operation that torch does not see either."""
    from torch.autograd import forward_ad
    from usaf_amd import few
    monkeypatch.setattr(fp8, "_linear", lambda x, w: torch.from_numpy(x.detach().as_subclass(torch.Tensor).float().numpy() * 3))
    monkeypatch.setattr(few, "_layer", lambda x, *_: torch.from_numpy(x.detach().as_subclass(torch.Tensor).float().numpy() * 3))
    x = torch.ones(2, 128, dtype=torch.bfloat16)
    ew, w, router = ExpertWeights(_t(2, 256, 128), _t(2, 128, 128)), _t(64, 128), torch.ones(2, 128, dtype=torch.bfloat16)

    def f(v, r=router):
        v = v.as_subclass(_OnGpu)
        return fp8.fp8_linear(v, w) if call == "linear" else few.few_token_block(v, r, 1, True, ew)

    with torch.no_grad():
        assert torch.equal(f(x).as_subclass(torch.Tensor), 3 * x.float())
    with forward_ad.dual_level():
        for args in [(forward_ad.make_dual(x, x),)] + ([(x, forward_ad.make_dual(router, router))] if call == "few" else []):
            with pytest.raises((NotImplementedError, RuntimeError), match="forward"):
                f(*args)
