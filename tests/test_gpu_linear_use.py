"""The 4-bit product and the gated projection as programs use them: weights that change, graphs side by side, host threads,
passes repeated, offsets past 32 bits."""
import threading

import pytest
import torch

import linear_oracle as O
from usaf_amd.gated import gated_linear
from usaf_amd.q4 import q4_linear

pytestmark = pytest.mark.gpu


def _weight(rows, k, seed=0):
    from usaf_amd.moe import Q4Tensor
    parts = O.codes(rows, k, seed)
    return Q4Tensor(*(t.cuda() for t in parts), torch.Size((rows, k))), parts


def _x(m, k, dtype=torch.bfloat16, seed=1):
    return torch.randn(m, k, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def _check(y, x, parts, n, k, what):
    ref, off = O.product(x.double().cpu(), O.weight(*parts, n, k, y.dtype))
    O.within(y, ref, O.rounded(ref, off, y.dtype), what)


@pytest.mark.parametrize("m", [1, 40, 600])
def test_a_weight_that_changes(m):
    n, k = 160, 384
    w, (q, s, z) = _weight(n, k)
    x = _x(m, k)
    _check(q4_linear(x, w), x, (q, s, z), n, k, "as made")
    w.s.mul_(2)  # in place
    _check(q4_linear(x, w), x, (q, s * 2, z), n, k, "scales doubled")
    w.z = (z * 4).cuda()  # another tensor
    _check(q4_linear(x, w), x, (q, s * 2, z * 4), n, k, "other zeros")
    w.q.copy_(q.flip(0))
    _check(q4_linear(x, w), x, (q.flip(0), s * 2, z * 4), n, k, "other codes")
    before = gated_linear(x, w)
    w.s.mul_(0.5)
    after = gated_linear(x, w)
    _, _, (act, off) = O.gated(x.double().cpu(), O.weight(q.flip(0), s, z * 4, n, k, x.dtype))
    O.within(after, act, O.rounded(act, off, x.dtype), "gated")
    assert not torch.equal(before, after)


def test_copies_of_a_weight():
    import copy
    import dataclasses
    n, k = 160, 384
    w, (q, s, z) = _weight(n, k)
    x = _x(40, k)
    _check(q4_linear(x, w), x, (q, s, z), n, k, "as made")
    other = dataclasses.replace(w, s=(s * 2).cuda())
    _check(q4_linear(x, other), x, (q, s * 2, z), n, k, "replaced")
    same = copy.copy(w)
    same.z = (z * 4).cuda()
    _check(q4_linear(x, same), x, (q, s, z * 4), n, k, "copied")
    _check(q4_linear(x, w), x, (q, s, z), n, k, "the first one")


def test_weights_and_rows_made_in_inference_mode():
    n, k = 64, 256
    with torch.inference_mode():
        w, parts = _weight(n, k)
        x = _x(9, k)
        y = q4_linear(x, w)
        act = gated_linear(x, w)
    _check(y, x, parts, n, k, "out")
    assert act.shape == (9, n // 2)


def test_passes_repeated_over_one_graph():
    w, _ = _weight(200, 256)
    dense = _x(180, 256, seed=5).mul(0.1).requires_grad_()
    x = _x(130, 256).requires_grad_()
    for y, leaves in ((q4_linear(x, w), (x,)), (gated_linear(x, w, "fp8"), (x,)), (gated_linear(x, dense, "fp8"), (x, dense)),
                      (gated_linear(x, dense), (x, dense))):
        dy = torch.ones_like(y[:1, :1]).expand_as(y)  # strides of zero
        first = torch.autograd.grad(y, leaves, dy, retain_graph=True)
        again = torch.autograd.grad(y, leaves, dy)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_the_same_rows_and_weight_twice_in_a_sum():
    w, _ = _weight(96, 128)
    x = _x(40, 128).requires_grad_()
    one = torch.autograd.grad(q4_linear(x, w).float().sum(), x)[0]
    two = torch.autograd.grad((q4_linear(x, w) + q4_linear(x, w)).float().sum(), x)[0]
    assert torch.equal(two, one * 2)


def test_two_host_threads():
    w, parts = _weight(512, 1024)
    dense = _x(256, 1024, seed=8).mul(0.05)
    xs = [_x(m, 1024, seed=m) for m in (3, 70, 400, 900)]
    want = [(q4_linear(x, w), gated_linear(x, w), gated_linear(x, dense)) for x in xs]
    torch.cuda.synchronize()
    bad, failed = [], []

    def work(stream):
        try:
            with torch.cuda.stream(stream):
                for _ in range(10):
                    for x, ys in zip(xs, want):
                        xg = x.clone().requires_grad_()
                        got = (q4_linear(x, w), gated_linear(x, w), gated_linear(x, dense))
                        gated_linear(xg, w, "fp8").backward(ys[1])
                        bad.extend(1 for a, b in zip(got, ys) if not torch.equal(a, b))
                stream.synchronize()
        except Exception as e:  # (told to the test's own thread)
            failed.append(e)

    threads = [threading.Thread(target=work, args=(torch.cuda.Stream(),)) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed and not bad


def test_two_graphs_side_by_side():
    """Each capture has workspaces of its own: replays on two streams do not meet in them."""
    w, _ = _weight(1024, 2048)
    big, _ = _weight(4096, 1024, seed=3)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    runs = []
    for i, st in enumerate(streams):
        x, xb = _x(100, 2048, seed=10 + i), _x(1500, 1024, seed=20 + i)
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            q4_linear(x, w), gated_linear(xb, big)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=st):
                out = (q4_linear(x, w), gated_linear(xb, big))
        runs.append((graph, x, xb, out))
    for n in range(4):
        for i, (_, x, xb, _) in enumerate(runs):
            x.copy_(_x(100, 2048, seed=30 + 2 * n + i))
            xb.copy_(_x(1500, 1024, seed=50 + 2 * n + i))
        torch.cuda.synchronize()
        for (graph, *_), st in zip(runs, streams):
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        for _, x, xb, out in runs:
            assert torch.equal(out[0], q4_linear(x, w)) and torch.equal(out[1], gated_linear(xb, big))


@pytest.mark.parametrize("m", [16, 1100])
def test_rows_far_apart(m):
    n, k, ld = 192, 256, 1 << 22
    if m * ld * 2 > torch.cuda.mem_get_info()[0] // 2:
        pytest.skip("not enough memory")
    w, parts = _weight(n, k)
    x = _x(m, k)
    far = torch.empty(m, ld, dtype=x.dtype, device="cuda")[:, :k]
    far.copy_(x)
    assert torch.equal(q4_linear(far, w), q4_linear(x, w))
    assert torch.equal(gated_linear(far, w), gated_linear(x, w))


def test_results_past_4_gib():
    """Rows at both ends of outputs, kept values and workspaces of more than 4 GiB."""
    m, inter, k = 70000, 32768, 128
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("not enough memory")
    gen = torch.Generator("cuda").manual_seed(0)
    x = torch.randn(m, k, generator=gen, device="cuda").bfloat16()
    dact = torch.randn(m, inter, generator=gen, device="cuda").bfloat16()
    w, parts = _weight(2 * inter, k)
    rows = torch.tensor([0, 1, 31999, 32768, m - 2, m - 1])
    xr = x[rows].double().cpu()
    _check(q4_linear(x, w)[rows], xr, parts, 2 * inter, k, "product")
    w64 = O.weight(*parts, 2 * inter, k, x.dtype)
    (g, off_g), (u, off_u), (act, off) = O.gated(xr, w64)
    dense = w64.to(x.dtype).cuda().requires_grad_()
    for weight, checkpoint in ((w, "fp8"), (dense, None)):
        xg = x.clone().requires_grad_()
        y = gated_linear(xg, weight, checkpoint)
        O.within(y.detach()[rows], act, O.rounded(act, off, x.dtype), "act")
        grads = torch.autograd.grad(y, (xg,) if checkpoint else (xg, dense), dact)
        # what is kept is within half a step (8 bits: of 4 significant ones, of the block's scale at least) of gate and up:
        # a few rows' gradient in the large call is the one that a call of these rows has, up to the sums' order
        few = x[rows].clone().requires_grad_()
        ref = torch.autograd.grad(gated_linear(few, weight, checkpoint), few, dact[rows])[0].double().cpu()
        # (dG, dU are the same up to ties of what is kept that the sums' order may turn: their share of a row's sum of
        # magnitudes is far below the tenth that a wrong row would miss it by)
        assert float((grads[0][rows].double().cpu() - ref).norm() / ref.norm()) < 0.02, "dx"
        assert torch.isfinite(grads[0]).all()
        if not checkpoint:
            cols = torch.tensor([0, 5, inter - 1, inter, 2 * inter - 1])
            at = cols % inter
            gd = x.double() @ dense.detach()[at].double().t()
            ud = x.double() @ dense.detach()[at + inter].double().t()
            (dg, _), (du, _) = O.gated_grads(dact[:, at].double(), gd.bfloat16().double(), ud.bfloat16().double())
            dgu = torch.where((cols < inter).cuda()[None, :], dg, du)
            want = (dgu.t() @ x.double()).cpu()
            bound = (dgu.abs().t() @ x.double().abs()).cpu() * (2.0 ** -8 * 2 + m * O.SUM)
            assert bool(((grads[1][cols].double().cpu() - want).abs() <= bound).all()), "dW"
        del y, grads, xg
