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
