"""Gate and up projection of a feed-forward layer with its gated activation, forward and backward.

``gated_linear`` is one expert's first half (usaf/qwen3moe_dml.py:58-61) for a dense layer or a
shared expert: act = silu(x Wg^T) * (x Wu^T) in one kernel, on a frozen 4-bit
``moe.Q4Tensor`` or a trained 16-bit weight.  A layer is completed by its down
projection, ``q4.q4_linear(gated_linear(x, gate_up), down)`` where it is 4-bit.

Rounding: gate and up are summed in fp32 and not rounded in front of the activation,
which is rounded once (the routed layer, which follows the reference's 16-bit tensors,
rounds gate, up, silu and their product).  For the backward they are kept in the activations'
dtype, 4 I bytes a token, or with ``checkpoint="fp8"`` in the 8-bit block format of
``fp8`` (e4m3 codes, a power-of-two scale for each 128 columns of gate and of up), 2.02 I:
there the gradients carry the 4 significant bits' error of gate and up (about 2.6 % of a value),
the output does not.  dG and dU are rounded to the activations' dtype, the products' operands.
"""
from __future__ import annotations

import functools
from typing import Optional, Union

import torch

from . import _native as N
from .fp8 import on
from .moe import Q4Tensor
from .q4 import Reading, _ld, check_weight, refuse_misfit, rows_of, words

CHECKPOINTS = (None, "fp8")


@functools.lru_cache(maxsize=4096)
def _ws_bytes(device: int, m: int, inter: int, k: int, four_bit: int, what: int) -> int:
    """The workspace on a device (its CU count decides the split), which is the current one."""
    return N.load().usaf_hip_gated_ws_bytes(m, inter, k, four_bit, what)


def _dense(w: torch.Tensor) -> torch.Tensor:
    w = w.contiguous()
    return w if w.data_ptr() % 16 == 0 else w.clone()


def _forward(x: torch.Tensor, w, checkpoint: Optional[str], keep: bool, read: Optional[Reading] = None):
    """act [M, I], and what the backward reads (None where nothing is kept): values and scales.  read: a 4-bit w's Reading, if
    there is one."""
    rows, k = (int(d) for d in w.shape)
    inter, m, dev = rows // 2, x.shape[0], x.device
    act = torch.empty(m, inter, dtype=x.dtype, device=dev)
    kept = scales = None
    if keep and checkpoint is None:
        kept = torch.empty(m, 2, -(-inter // 8) * 8, dtype=x.dtype, device=dev)
    elif keep:
        blocks = -(-inter // 128)
        kept = torch.empty(m, 2, blocks * 128, dtype=torch.uint8, device=dev)
        scales = torch.empty(m, 2, blocks, dtype=torch.uint8, device=dev)
    if m:
        if isinstance(w, Q4Tensor):  # (codes, scale words, 16-bit weight), held until the launch
            parts = (w.q, words("gated_linear", w), None) if read is None else (read.q, read.sz, None)
        else:
            parts = (None, None, w)
        with on(dev):
            need = _ws_bytes(dev.index, m, inter, k, int(isinstance(w, Q4Tensor)), 0 if scales is None else 4)
            ws = torch.empty(need, dtype=torch.uint8, device=dev) if need > 0 else None
            N.call("usaf_hip_gated_fwd", x.data_ptr(), N.dtype_code(x.dtype), m, k, _ld(x), *map(N.ptr, parts), inter,
                   act.data_ptr(), N.ptr(kept), N.ptr(scales), N.ptr(ws), max(need, 0), N.stream_ptr(dev))
    return act, kept, scales


class GatedLinearFn(torch.autograd.Function):
    """act = silu(x Wg^T) (x Wu^T) of rows x [M, K]; w is the weight, trained where it is a tensor that wants a gradient.
    checked: the caller has looked at them (a trace calls this by itself)."""

    @staticmethod
    def forward(ctx, x: torch.Tensor, weight: Optional[torch.Tensor], q4: Optional[Q4Tensor], checkpoint: Optional[str],
                checked: bool):
        keep = any(ctx.needs_input_grad[:2])
        if not checked:
            if q4 is not None:
                check_weight("gated_linear", q4)
            refuse_misfit("gated_linear", x, weight if q4 is None else q4)
        read = None if q4 is None else Reading.of("gated_linear", q4, x)
        rows = rows_of(x, x.shape[1])
        w = q4 if weight is None else _dense(weight)
        act, kept, scales = _forward(rows, w, checkpoint, keep, read)
        ctx.dtype, ctx.shape = x.dtype, tuple(w.shape)
        if keep:
            ctx.read = read
            ctx.save_for_backward(kept, scales, x if ctx.needs_input_grad[1] else None,
                                  weight if ctx.needs_input_grad[0] else None)
        return act

    @staticmethod
    def backward(ctx, dact: torch.Tensor):
        if torch.is_grad_enabled():
            raise RuntimeError("gated_linear has no second derivative (create_graph=True)")
        N.refuse_capture("gated_linear's backward")
        if ctx.read is not None:
            ctx.read.refuse_written("gated_linear's backward")
        want_x, want_w = ctx.needs_input_grad[:2]
        kept, scales, x, weight = ctx.saved_tensors
        (rows, k), (m, dev) = ctx.shape, (dact.shape[0], dact.device)
        dx = torch.empty(m, k, dtype=ctx.dtype, device=dev) if want_x else None
        dw = torch.empty(rows, k, dtype=ctx.dtype, device=dev) if want_w else None
        if m == 0:
            return dx, None if dw is None else dw.zero_(), None, None, None
        dact = dact.to(ctx.dtype).contiguous()
        # (a saved-tensor hook may have changed what was kept: its layout, its place)
        kept, scales = _dense(kept), None if scales is None else scales.contiguous()
        if ctx.read is not None:
            parts = (ctx.read.q, ctx.read.sz, None)
        else:  # only dx reads the weight; without it any 16-bit pointer says that there is no 4-bit one
            parts = (None, None, kept if weight is None else _dense(weight))
        if want_w:
            x = rows_of(x, k)
        with on(dev):
            need = _ws_bytes(dev.index, m, rows // 2, k, int(ctx.read is not None), int(want_x) + 2 * int(want_w))
            ws = torch.empty(max(need, 0), dtype=torch.uint8, device=dev)
            N.call("usaf_hip_gated_bwd", dact.data_ptr(), N.dtype_code(ctx.dtype), m, rows // 2, k, kept.data_ptr(),
                   N.ptr(scales), *map(N.ptr, parts), x.data_ptr() if want_w else None, _ld(x) if want_w else k, N.ptr(dx),
                   N.ptr(dw), ws.data_ptr(), ws.numel(), N.stream_ptr(dev))
        return dx, dw, None, None, None


def gated_linear(x: torch.Tensor, gate_up: Union[Q4Tensor, torch.Tensor], checkpoint: Optional[str] = None) -> torch.Tensor:
    """x [..., K] fp16 / bf16, gate_up [2 I, K] (the gate's rows, then up's) -> silu(gate) * up
    [..., I] in x's dtype.

    gate_up: a ``Q4Tensor`` (group size 128 along whole rows), frozen, or a tensor of x's
    dtype, which receives a gradient where it wants one.  checkpoint: None keeps gate and up
    in x's dtype for the backward, "fp8" in 8-bit blocks; without a gradient nothing is kept.
    No second or forward-mode derivatives; torch.jit.trace records the call.  A stream
    capture takes calls without a gradient only, of 4-bit weights once they have been used.
    What is said of a weight's writes and lifetime at ``q4_linear`` holds here."""
    if checkpoint not in CHECKPOINTS:
        raise ValueError(f"gated_linear: checkpoint must be one of {CHECKPOINTS}, got {checkpoint!r}")
    four_bit = isinstance(gate_up, Q4Tensor)
    if four_bit:
        check_weight("gated_linear", gate_up)
    elif not isinstance(gate_up, torch.Tensor):
        raise TypeError(f"gated_linear: gate_up must be a Q4Tensor or a tensor, got {type(gate_up).__name__}")
    shape = tuple(int(d) for d in gate_up.shape)
    if len(shape) != 2 or shape[0] < 2 or shape[0] % 2 or shape[1] < 1:
        raise ValueError(f"gated_linear: need a weight [2 I, K], got {shape}")
    refuse_misfit("gated_linear", x, gate_up)
    rows = x if x.dim() == 2 else x.reshape(x.numel() // shape[1], shape[1])
    grad = torch.is_grad_enabled() and (x.requires_grad or (not four_bit and gate_up.requires_grad))
    if grad:
        N.refuse_capture("gated_linear of tensors that want a gradient")
    if grad or N.followed(x, *(() if four_bit else (gate_up,))):
        weight, q4 = (None, gate_up) if four_bit else (gate_up, None)
        act = GatedLinearFn.apply(rows, weight, q4, checkpoint, grad and not torch.jit.is_tracing())
    else:
        act = _forward(rows_of(rows, shape[1]), gate_up if four_bit else _dense(gate_up), checkpoint, False)[0]
    return act if x.dim() == 2 else act.view(*x.shape[:-1], shape[0] // 2)
