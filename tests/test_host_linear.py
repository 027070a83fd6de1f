"""Argument checks of the 4-bit product and the gated projection: no GPU work."""
import ctypes

import pytest
import torch

import linear_oracle as O
from usaf_amd import _native as N
from usaf_amd.gated import gated_linear
from usaf_amd.moe import Q4Tensor
from usaf_amd.q4 import q4_linear


def _w(rows, k, **change):
    q, s, z = O.codes(rows, k)
    parts = {"q": q, "s": s, "z": z, "shape": torch.Size((rows, k)), **change}
    return Q4Tensor(parts["q"], parts["s"], parts["z"], parts["shape"], parts.get("group_size", 128))


@pytest.mark.parametrize("call", [q4_linear, gated_linear])
def test_refusals(call):
    x = torch.zeros(3, 256, dtype=torch.bfloat16)
    w = _w(64, 256)
    with pytest.raises(ValueError, match="GPU"):
        call(x, w)
    with pytest.raises(ValueError, match="fit"):
        call(x[:, :128], w)
    with pytest.raises(ValueError, match="fit"):
        call(torch.zeros((), dtype=torch.bfloat16), w)
    with pytest.raises(TypeError, match="fp16 or bf16"):
        call(x.float(), w)
    with pytest.raises(ValueError, match="weight"):
        call(x, _w(64, 256, shape=torch.Size((1, 64, 256))))
    with pytest.raises(NotImplementedError, match="dequantize"):
        call(x, _w(64, 256, group_size=64))
    with pytest.raises(NotImplementedError):
        call(x, _w(128, 128, shape=torch.Size((64, 192))))
    q = O.codes(64, 256)[0]
    for change in [{"q": q[:-1]}, {"q": q.view(-1, 32)}, {"s": torch.zeros(3).half()}, {"q": q.t().contiguous().t()},
                   {"q": torch.zeros(q.numel() + 1, dtype=torch.int8)[1:].view_as(q)}]:
        with pytest.raises(ValueError):
            call(x, _w(64, 256, **change))
    with pytest.raises(TypeError):
        call(x, _w(64, 256, s=torch.zeros(128)))
    with pytest.raises(TypeError):
        call(x, _w(64, 256, q=q.short()))


def test_gated_refusals():
    x, w = torch.zeros(3, 100, dtype=torch.float16), torch.zeros(64, 100, dtype=torch.float16)
    with pytest.raises(ValueError, match="GPU"):
        gated_linear(x, w)
    with pytest.raises(ValueError, match="checkpoint"):
        gated_linear(x, w, checkpoint="int8")
    with pytest.raises(TypeError, match="dtype"):
        gated_linear(x, w.float())
    with pytest.raises(TypeError, match="Q4Tensor or a tensor"):
        gated_linear(x, [w])
    for bad in [w[:63], w[0], w[:0], w[None]]:
        with pytest.raises(ValueError, match="2 I"):
            gated_linear(x, bad)
    with pytest.raises(ValueError, match="2 I"):
        gated_linear(torch.zeros(3, 128, dtype=torch.float16), _w(63, 128))


def test_entry_points_check_their_arguments():
    lib, p, odd, even = N.load(), ctypes.c_void_p(4096), ctypes.c_void_p(4097), ctypes.c_void_p(4098)
    inval, ok, unsup = N.USAF_ERR_INVALID, N.USAF_OK, N.USAF_ERR_UNSUPPORTED
    big = 1 << 40

    def linear(name="usaf_hip_q4_linear", x=p, dtype=N.BF16, m=4, cols=256, ld=256, q=p, sz=p, other=64, out=p, ws=p, size=big):
        return getattr(lib, name)(x, dtype, m, cols, ld, q, sz, other, out, ws, size, None)

    assert linear(m=0, x=None, q=None, sz=None, out=None, ws=None, size=0) == ok
    for bad in [dict(m=-1), dict(m=1 << 31), dict(cols=0), dict(cols=100), dict(cols=1 << 23), dict(other=0), dict(other=1 << 23),
                dict(dtype=N.F32), dict(x=None), dict(q=None), dict(sz=None), dict(out=None), dict(ld=255), dict(ld=1 << 23),
                dict(ld=257), dict(q=even), dict(sz=even), dict(x=even), dict(out=odd), dict(m=4096, other=4096, ws=None),
                dict(m=4096, other=4096, size=100), dict(m=4096, other=4096, ws=even)]:
        assert linear(**bad) == inval, bad
    assert "q4_linear" in N.last_error()
    back = dict(name="usaf_hip_q4_linear_bwd", cols=64, ld=64, other=256)
    for bad in [dict(other=100), dict(ws=None), dict(size=10), dict(x=even), dict(cols=63, ld=62), dict(dtype=7)]:
        assert linear(**{**back, **bad}) == inval, bad
    assert linear(**{**back, "m": 0}) == ok

    def fwd(x=p, dtype=N.F16, m=4, k=256, ld=256, q=p, sz=p, w16=None, inter=32, act=p, kept=None, scales=None, ws=p, size=big):
        return lib.usaf_hip_gated_fwd(x, dtype, m, k, ld, q, sz, w16, inter, act, kept, scales, ws, size, None)

    assert fwd(m=0, x=None, q=None, sz=None, act=None, ws=None, size=0) == ok
    for bad in [dict(m=-1), dict(inter=0), dict(inter=1 << 22), dict(k=0), dict(k=192), dict(dtype=N.F32), dict(q=None),
                dict(w16=p), dict(sz=None), dict(q=even), dict(sz=even), dict(q=None, sz=None, w16=even), dict(x=None),
                dict(act=None), dict(act=odd), dict(x=even), dict(ld=200), dict(ld=260), dict(scales=p), dict(kept=even),
                dict(q=None, sz=None, w16=p, k=100, ld=100, ws=None), dict(q=None, sz=None, w16=p, k=100, ld=100, size=64),
                dict(m=4096, inter=4096, ws=even)]:
        assert fwd(**bad) == inval, bad
    assert fwd(inter=1 << 20, k=1 << 14, ld=1 << 14) == unsup

    def bwd(dact=p, dtype=N.F16, m=4, inter=32, k=256, kept=p, scales=None, q=None, sz=None, w16=p, x=p, ldx=256, dx=p, dw=p,
            ws=p, size=big):
        return lib.usaf_hip_gated_bwd(dact, dtype, m, inter, k, kept, scales, q, sz, w16, x, ldx, dx, dw, ws, size, None)

    assert bwd(m=0) == ok
    for bad in [dict(m=-1), dict(dtype=N.F32), dict(w16=None), dict(q=p, sz=p), dict(q=p, sz=p, w16=None), dict(dact=None),
                dict(kept=None), dict(dx=None, dw=None), dict(x=None), dict(ldx=100), dict(kept=even), dict(dact=odd), dict(dw=odd),
                dict(ws=None), dict(size=100), dict(m=1 << 23)]:
        assert bwd(**bad) == inval, bad


def test_workspace_sizes():
    lib = N.load()
    sizes, gated = lib.usaf_hip_q4_linear_ws_bytes, lib.usaf_hip_gated_ws_bytes
    for bad in [(-1, 64, 128, 0), (1, 0, 128, 0), (1, 64, 0, 0), (1, 1 << 23, 128, 0), (1 << 31, 64, 128, 0)]:
        assert sizes(*bad) == -1
    for bad in [(-1, 64, 128, 0, 0), (1, 0, 128, 0, 0), (1, 64, 128, 0, 5), (1, 64, 128, 0, -1), (1, 1 << 22, 128, 0, 0)]:
        assert gated(*bad) == -1
    assert sizes(1, 4096, 4096, 0) == 0 and gated(1, 4096, 4096, 1, 0) == 0
    for m in (0, 1, 700):  # more is wanted, more is needed
        assert 0 <= gated(m, 100, 130, 0, 1) <= gated(m, 100, 130, 0, 3) <= gated(m + 64, 100, 130, 0, 3)
        assert 0 <= sizes(m, 100, 128, 1) <= sizes(m + 1, 100, 128, 1)


def test_formulas_by_differences():
    """The oracle's gradients against differences of its own activation, in 64 bits."""
    gen = torch.Generator().manual_seed(0)
    x, w, d = (torch.randn(*s, dtype=torch.float64, generator=gen) for s in [(5, 7), (12, 7), (5, 6)])
    (g, _), (u, _), _ = O.gated(x, w)
    (dg, _), (du, _) = O.gated_grads(d, g, u)
    dgu = torch.cat([dg, du], 1)
    h = 1e-6
    for grad, t in ((dgu @ w, x), (dgu.t() @ x, w)):
        for at in range(0, t.numel(), 3):
            value = []
            for sign in (1, -1):
                t.view(-1)[at] += sign * h
                value.append(float((O.gated(x, w)[2][0] * d).sum()))
                t.view(-1)[at] -= sign * h
            assert abs((value[0] - value[1]) / (2 * h) - float(grad.reshape(-1)[at])) < 1e-6 * (1 + abs(float(grad.reshape(-1)[at])))
