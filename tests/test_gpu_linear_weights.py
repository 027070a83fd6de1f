"""4-bit weights of the product and the gated projection that are written to or replaced: made in inference mode, between
a forward and its backward, beside a call that reads them."""
import pytest
import torch

import linear_oracle as O
import test_gpu_linear_use as U
from usaf_amd.gated import gated_linear
from usaf_amd.q4 import q4_linear

pytestmark = pytest.mark.gpu
N_, K = 160, 384


def _check_gated(y, x, parts, what):
    _, _, (act, off) = O.gated(x.double().cpu(), O.weight(*parts, N_, K, y.dtype))
    O.within(y, act, O.rounded(act, off, y.dtype), what)


@pytest.mark.parametrize("m", [1, 40, 600])
@pytest.mark.parametrize("which", ["s", "z", "both"])
def test_writes_to_a_weight_made_in_inference_mode(m, which):
    """Torch counts no writes to such tensors: the scale words follow them all the same."""
    w, (q, s, z) = U._weight(N_, K)
    x = U._x(m, K)
    with torch.inference_mode():
        if which != "z":
            w.s = s.cuda()
        if which != "s":
            w.z = z.cuda()
        U._check(q4_linear(x, w), x, (q, s, z), N_, K, "as made")
        _check_gated(gated_linear(x, w), x, (q, s, z), "gated, as made")
        if which != "z":
            w.s.mul_(2)
            s = s * 2
        if which != "s":
            w.z.mul_(4)
            z = z * 4
        U._check(q4_linear(x, w), x, (q, s, z), N_, K, "written to")
        _check_gated(gated_linear(x, w), x, (q, s, z), "gated, written to")
        w.q.copy_(q.flip(0))
        U._check(q4_linear(x, w), x, (q.flip(0), s, z), N_, K, "other codes")
    U._check(q4_linear(x, w), x, (q.flip(0), s, z), N_, K, "outside of inference mode")


@pytest.mark.parametrize("m", [1, 600])
def test_a_graph_over_a_weight_made_in_inference_mode(m):
    """The words are the capture's own, made anew by each replay."""
    x = U._x(m, K)
    with torch.inference_mode():
        w, (q, s, z) = U._weight(N_, K)
        q4_linear(x, w), gated_linear(x, w)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y, act = q4_linear(x, w), gated_linear(x, w)
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            U._check(y, x, (q, s, z), N_, K, "replayed")
            _check_gated(act, x, (q, s, z), "gated, replayed")
            w.s.mul_(2)
            s = s * 2
            assert torch.equal(q4_linear(x, w), q4_linear(x.clone(), w))


CALLS = {"linear": q4_linear, "gated": gated_linear, "checkpoint": lambda x, w: gated_linear(x, w, "fp8")}


def _leaf(m):
    return U._x(m, K).requires_grad_()


@pytest.mark.parametrize("m", [1, 40, 600])
@pytest.mark.parametrize("call", list(CALLS))
@pytest.mark.parametrize("part", ["q", "s", "z"])
def test_a_weight_written_to_before_its_backward(call, part, m):
    """As torch does for a tensor that a backward needs."""
    w, _ = U._weight(N_, K)
    y = CALLS[call](_leaf(m), w)
    t = getattr(w, part)
    t.copy_(t.flip(0))
    with pytest.raises(RuntimeError, match="written to"):
        y.float().sum().backward()
    with torch.no_grad():
        CALLS[call](U._x(m, K), w)  # (lays the scale words out anew)
    with pytest.raises(RuntimeError, match="written to"):
        CALLS[call](_leaf(m), w)
        y.float().sum().backward()


@pytest.mark.parametrize("made", ["as usual", "in inference mode"])
@pytest.mark.parametrize("m", [1, 40, 600])
@pytest.mark.parametrize("call", list(CALLS))
def test_a_weight_given_other_tensors_before_its_backward(call, m, made):
    """The gradient is that of the weight that the forward read, also where another forward has read the new one."""
    with torch.inference_mode(made != "as usual"):
        w, _ = U._weight(N_, K, seed=1)
        other, _ = U._weight(N_, K, seed=2)
    x = _leaf(m)
    dy = torch.ones_like(CALLS[call](x, w))
    want = torch.autograd.grad(CALLS[call](x, w), x, dy)[0]
    for between in (False, True):
        y = CALLS[call](x, w)
        old = w.q, w.s, w.z
        w.q, w.s, w.z = other.q, other.s, other.z
        z = CALLS[call](x, w) if between else None
        assert torch.equal(torch.autograd.grad(y, x, dy, retain_graph=True)[0], want)
        assert torch.equal(torch.autograd.grad(y, x, dy)[0], want)
        if between:
            new = torch.autograd.grad(CALLS[call](x, other), x, dy)[0]
            assert torch.equal(torch.autograd.grad(z, x, dy)[0], new) and not torch.equal(new, want)
        w.q, w.s, w.z = old


def test_calls_of_no_rows_need_no_words():
    """Also in a capture, on a weight that has not been used."""
    w, _ = U._weight(N_, K)
    x = torch.empty(0, K, dtype=torch.bfloat16, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph), torch.no_grad():
        assert q4_linear(x, w).shape == (0, N_) and gated_linear(x, w).shape == (0, N_ // 2)
    x = x.clone().requires_grad_()
    (q4_linear(x, w).sum() + gated_linear(x, w).sum()).backward()
    assert x.grad.shape == (0, K) and w._szg is None


@pytest.mark.parametrize("call", list(CALLS))
def test_a_trace_over_a_weight_that_is_written_to(call):
    """A recorded call reads the weight as a call does."""
    w, _ = U._weight(N_, K)
    x = U._x(40, K)
    traced = torch.jit.trace(lambda t: CALLS[call](t, w), (x,), check_trace=False)
    before = traced(x)
    assert torch.equal(before, CALLS[call](x, w))
    w.s.mul_(2)
    after = traced(x)
    assert not torch.equal(before, after) and torch.equal(after, CALLS[call](x, w))
    w.z = w.z * 2
    again = traced(x)
    assert not torch.equal(again, after) and torch.equal(again, CALLS[call](x, w))


def test_a_trace_refuses_what_a_call_refuses():
    """Other rows than the traced ones are not read past their end or as another type."""
    w, _ = U._weight(N_, K)
    dense = U._x(N_, K, seed=3)
    x = U._x(40, K)
    for call, weight in ((q4_linear, w), (gated_linear, w), (gated_linear, dense)):
        traced = torch.jit.trace(lambda t: call(t, weight), (x,), check_trace=False)
        assert torch.equal(traced(x[:7]), call(x[:7], weight))
        for bad in (torch.cat([x, x], 1), x[:, :256], x.cpu(), x.float()):
            with pytest.raises((ValueError, TypeError, RuntimeError)):
                traced(bad)
        if weight is dense:
            with pytest.raises((ValueError, TypeError, RuntimeError)):
                traced(x.half())
        else:
            assert torch.equal(traced(x.half()), call(x.half(), weight))


@pytest.mark.parametrize("part", ["q", "s", "z"])
def test_a_weight_whose_tensors_are_given_other_memory(part):
    """``t.data = other``: t is the same object, and torch counts no write."""
    w, (q, s, z) = U._weight(N_, K)
    x, leaf = U._x(40, K), _leaf(40)
    U._check(q4_linear(x, w), x, (q, s, z), N_, K, "as made")
    y = q4_linear(leaf, w)
    parts = {"q": q, "s": s, "z": z}
    parts[part] = parts[part].flip(0)
    getattr(w, part).data = parts[part].cuda()
    U._check(q4_linear(x, w), x, tuple(parts.values()), N_, K, "other memory")
    _check_gated(gated_linear(x, w), x, tuple(parts.values()), "gated, other memory")
    with pytest.raises(RuntimeError, match="written to"):
        y.float().sum().backward()
    getattr(w, part).data = parts[part][:-1].cuda()
    for call in CALLS.values():
        with pytest.raises(ValueError, match="fit"):
            call(x, w)
