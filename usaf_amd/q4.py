"""The product with one 4-bit weight.

``q4_linear`` is ``F.linear`` with a ``moe.Q4Tensor`` of shape [N, K], as
``quantize_4bit`` makes it (group size 128 along whole rows), beside ``fp8.fp8_linear``:
a projection or an output head that is kept in 4 bits, for one token or a prompt,
differentiable in the activations.  Calls of a few hundred rows or more, and every
backward, write the weight's 16-bit values to a workspace of their own.  A weight's value is everywhere the
codec's in the activations' dtype, ``w.dequantize(x.dtype)`` bit for bit
(fp16(code * scale) + zero in fp16, usaf/quantization.py:88-132, then bf16 where
the activations are), so decoding, prompts and gradients multiply the same numbers.
"""
from __future__ import annotations

import functools
from typing import NamedTuple, Optional

import torch

from . import _native as N
from .fp8 import on
from .moe import Q4Tensor

ACT = (torch.float16, torch.bfloat16)
MAX_COLS = 1 << 22


@functools.lru_cache(maxsize=4096)
def _ws_bytes(device: int, m: int, n: int, k: int, backward: int) -> int:
    """The workspace on a device (its CU count decides the split), which is the current one."""
    return N.load().usaf_hip_q4_linear_ws_bytes(m, n, k, backward)


def _versions(*tensors: torch.Tensor):
    """Where tensors lie (``t.data = other`` leaves t itself) and counts of the writes to them (None where made in inference
    mode, which counts none)."""
    return [(t.data_ptr(), None if t.is_inference() else t._version) for t in tensors]


def check_weight(what: str, w: Q4Tensor) -> None:
    """Raise unless w is a 4-bit matrix in the layout that the products read (looked at once for each set of tensors: 5 us)."""
    seen, now = w.__dict__.get("_seen"), (w.shape, w.group_size, w.q.data_ptr(), _versions(w.s, w.z))
    if seen is not None and seen[0] is w.q and seen[1] is w.s and seen[2] is w.z and seen[3] == now:
        return
    if len(w.shape) != 2 or any(int(d) < 1 for d in w.shape):
        raise ValueError(f"{what}: need a 4-bit weight [rows, K], got {tuple(w.shape)}")
    rows, k = (int(d) for d in w.shape)
    if w.group_size != 128 or k % 128:
        raise NotImplementedError(f"{what}: needs group size 128 along whole rows (K a multiple of 128), got {tuple(w.shape)}, "
                                  f"group size {w.group_size}; dequantize() takes any")
    groups = rows * k // 128
    if tuple(w.q.shape) != (groups, 64) or w.s.numel() != groups or w.z.numel() != groups:
        raise ValueError(f"{what}: codes {tuple(w.q.shape)}, scales {tuple(w.s.shape)} and zeros {tuple(w.z.shape)} do not fit "
                         f"{tuple(w.shape)}: need {(groups, 64)} and {groups} each")
    if w.q.element_size() != 1 or w.s.dtype != torch.float16 or w.z.dtype != torch.float16:
        raise TypeError(f"{what}: codes are bytes, scales and zeros fp16, got {w.q.dtype}, {w.s.dtype}, {w.z.dtype}")
    if not (w.q.is_contiguous() and w.s.is_contiguous() and w.z.is_contiguous()) or w.q.data_ptr() % 16 \
            or w.s.device != w.q.device or w.z.device != w.q.device:
        raise ValueError(f"{what}: codes, scales and zeros must be contiguous, on one device, the codes 16-byte aligned")
    w._szg = None  # (a copy of a tensor with other parts may have brought its words along)
    w.__dict__["_seen"] = (w.q, w.s, w.z, now)


def words(what: str, w: Q4Tensor) -> torch.Tensor:
    """The scale/zero words by group, int32 [K / 128, rows] (Q4Tensor.scale_zero_by_group's of one matrix): built once and
    kept with the weight, finished when built, so that any stream may read them from then on.  Of scales or zeros made in
    inference mode, whose writes nobody counts, they are the call's own instead, built on its stream, in a capture too."""
    szg = w._szg
    if szg is None or szg.device != w.device:
        kept = not (w.s.is_inference() or w.z.is_inference())
        if kept:
            N.refuse_capture(f"{what}: the first call on a weight")
        rows, k = (int(d) for d in w.shape)
        with on(w.device):
            by_row = torch.empty(rows, k // 128, dtype=torch.int32, device=w.device)
            N.call("usaf_hip_pack_scale_zero", w.s.data_ptr(), w.z.data_ptr(), by_row.numel(), by_row.data_ptr(),
                   N.stream_ptr(w.device))
            szg = by_row.t().contiguous()
            if kept:
                torch.cuda.current_stream(w.device).synchronize()
                w._szg = szg
    return szg


def refuse_misfit(what: str, x: torch.Tensor, w) -> None:
    """Raise unless x's rows can be multiplied by a weight [.., K], 4-bit or of x's own type, on its device."""
    if x.dtype not in ACT:
        raise TypeError(f"{what}: activations must be fp16 or bf16, got {x.dtype}")
    if not isinstance(w, Q4Tensor) and w.dtype != x.dtype:
        raise TypeError(f"{what}: a 16-bit weight must be of the activations' dtype, got {w.dtype} and {x.dtype}")
    if x.dim() < 1 or x.shape[-1] != w.shape[1]:
        raise ValueError(f"{what}: activations {tuple(x.shape)} do not fit the weight {tuple(w.shape)}")
    if x.device != w.device or not x.is_cuda:
        raise ValueError(f"{what}: activations on {x.device}, weight on {w.device}: both on one GPU")


class Reading(NamedTuple):
    """A weight's tensors as a forward reads them, which are what its backward reads, whatever the weight holds by then."""
    q: torch.Tensor
    s: torch.Tensor
    z: torch.Tensor
    sz: Optional[torch.Tensor]  # words() of s and z, None for a call of no rows
    versions: list

    @classmethod
    def of(cls, what: str, w: Q4Tensor, x: torch.Tensor) -> "Reading":
        return cls(w.q, w.s, w.z, words(what, w) if x.numel() else None, _versions(w.q, w.s, w.z))

    def refuse_written(self, what: str) -> None:
        """Raise, as for a torch tensor that a backward needs, where these have been written to since."""
        if _versions(self.q, self.s, self.z) != self.versions:
            raise RuntimeError(f"{what}: the 4-bit weight's codes, scales or zeros have been written to since the forward")


def rows_of(t: torch.Tensor, cols: int) -> torch.Tensor:
    """t as rows [M, cols] that start at multiples of 16 bytes, without a copy where they do."""
    t = t if t.dim() == 2 else t.reshape(t.numel() // cols, cols)
    if t.stride(1) != 1 or (t.shape[0] > 1 and not (cols <= t.stride(0) <= MAX_COLS and t.stride(0) % 8 == 0)):
        t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)


def _ld(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else -(-t.shape[1] // 8) * 8


class Q4LinearFn(torch.autograd.Function):
    """y = x W^T; dx = dy W.  checked: the caller has looked at x and w (a trace calls this by itself)."""

    @staticmethod
    def forward(ctx, x: torch.Tensor, w: Q4Tensor, checked: bool):
        if not checked:
            check_weight("q4_linear", w)
            refuse_misfit("q4_linear", x, w)
        read = Reading.of("q4_linear", w, x)
        if ctx.needs_input_grad[0]:
            ctx.read, ctx.shape, ctx.dtype = read, w.shape, x.dtype
        return _linear(x, w.shape, read.q, read.sz)

    @staticmethod
    def backward(ctx, dy: torch.Tensor):
        if torch.is_grad_enabled():
            raise RuntimeError("q4_linear has no second derivative (create_graph=True)")
        N.refuse_capture("q4_linear's backward")
        ctx.read.refuse_written("q4_linear's backward")
        dy = dy if dy.dtype == ctx.dtype else dy.to(ctx.dtype)
        return _linear(dy, ctx.shape, ctx.read.q, ctx.read.sz, backward=True), None, None


def _linear(x: torch.Tensor, shape, q: torch.Tensor, sz: Optional[torch.Tensor], backward: bool = False) -> torch.Tensor:
    n, k = (int(d) for d in shape)
    dev, (cols, out_cols) = x.device, (n, k) if backward else (k, n)
    rows = rows_of(x, cols)
    m = rows.shape[0]
    out = torch.empty(m, out_cols, dtype=x.dtype, device=dev)
    if m:
        with on(dev):
            need = _ws_bytes(dev.index, m, n, k, int(backward))
            ws = torch.empty(need, dtype=torch.uint8, device=dev) if need > 0 else None
            name, size = ("usaf_hip_q4_linear_bwd", k) if backward else ("usaf_hip_q4_linear", n)
            N.call(name, rows.data_ptr(), N.dtype_code(x.dtype), m, cols, _ld(rows), q.data_ptr(), sz.data_ptr(), size,
                   out.data_ptr(), N.ptr(ws), max(need, 0), N.stream_ptr(dev))
    return out if x.dim() == 2 else out.view(*x.shape[:-1], out_cols)


def q4_linear(x: torch.Tensor, w: Q4Tensor) -> torch.Tensor:
    """F.linear with a 4-bit weight: x [..., K] fp16 / bf16, w [N, K] -> [..., N] in x's
    dtype, summed in fp32 and rounded once.  Differentiable in x (the weight is
    frozen).  The first call on a weight builds its scale words (1/17 of it), not in
    a stream capture; a capture takes calls without a gradient only.  There is no
    forward-mode derivative; torch.jit.trace records the call.  Scales or zeros that torch
    has written to since are laid out again, but for writes through ``.data`` or by other
    kernels, which torch does not count; those made in inference mode, where it counts
    none, are laid out by every call (two more launches).  A weight is kept, and not written
    to, until the work that reads it, a graph's replays too, has ended.  A backward reads the
    forward's tensors, also where the weight has been given others since, and raises where
    torch has counted a write to them."""
    check_weight("q4_linear", w)
    refuse_misfit("q4_linear", x, w)
    if torch.is_grad_enabled() and x.requires_grad:
        N.refuse_capture("q4_linear of activations that want a gradient")
        return Q4LinearFn.apply(x, w, not torch.jit.is_tracing())
    if N.followed(x):
        return Q4LinearFn.apply(x, w, False)
    # (the function's own call takes 2 us of the host's time)
    return _linear(x, w.shape, w.q, words("q4_linear", w) if x.numel() else None)
