"""The scale words that a call hands to a kernel, on the CPU: no GPU work, the library's calls are watched instead."""
import contextlib
import weakref

import pytest
import torch

import linear_oracle as O
from usaf_amd import _native as N
from usaf_amd import gated, q4
from usaf_amd.moe import Q4Tensor


@pytest.fixture
def watched(monkeypatch):
    """A weight whose words another call drops as soon as a call has asked for them; notes whether what a launch gets lives."""
    w = Q4Tensor(*O.codes(64, 128), torch.Size((64, 128)))
    alive, made = [], []

    def words():
        w._szg = torch.zeros(1, 64, dtype=torch.int32)
        made.append(weakref.ref(w._szg))

    def dropped(*_):
        w._szg = None
        return 0

    def call(name, *args):
        alive.append((name, any(r() is not None and r().data_ptr() in args for r in made)))
        words()

    for module in (gated, q4):
        monkeypatch.setattr(module, "on", lambda _: contextlib.nullcontext())
        monkeypatch.setattr(module, "_ws_bytes", dropped)
    monkeypatch.setattr(N, "call", call)
    monkeypatch.setattr(N, "stream_ptr", lambda _: None)
    monkeypatch.setattr(N, "refuse_capture", lambda _: None)
    q4.check_weight("", w)
    words()
    return w, alive


def test_words_live_until_the_launch(watched):
    w, alive = watched
    x = torch.zeros(4, 128, dtype=torch.bfloat16, requires_grad=True)
    gated.GatedLinearFn.apply(x, None, w, None, True).sum().backward()
    q4.Q4LinearFn.apply(x, w, True).sum().backward()
    assert alive == [(f"usaf_hip_{name}", True) for name in ("gated_fwd", "gated_bwd", "q4_linear", "q4_linear_bwd")]


@pytest.mark.parametrize("call", [q4.q4_linear, gated.gated_linear])
def test_refusals_of_activations_that_want_a_gradient(call):
    """The same as without one."""
    w = Q4Tensor(*O.codes(64, 256), torch.Size((64, 256)))
    x = torch.zeros(3, 256, dtype=torch.bfloat16, requires_grad=True)
    with pytest.raises(ValueError, match="GPU"):
        call(x, w)
    with pytest.raises(ValueError, match="fit"):
        call(x[:, :128], w)
    with pytest.raises(ValueError, match="fit"):
        call(x[0, 0], w)
    with pytest.raises(TypeError, match="fp16 or bf16"):
        call(x.float(), w)
    with pytest.raises(NotImplementedError, match="dequantize"):
        call(x, Q4Tensor(w.q, w.s, w.z, w.shape, 64))
