"""8-bit block-scaled weights: the codec, the product and its grad-input.

Codes are e4m3; every block of 128 values (activations: 1 x 128 along the row,
weights: 128 x 128) has one power-of-two scale, held as the E8M0 byte e + 127
with e the smallest integer that brings the block's largest magnitude to 448 or
below.  The matrix instruction applies such scales itself, so a product reads
the codes as they are, where the 4-bit format's weights are first dequantized
by vector instructions.  A weight takes 1.00006 bytes an element.

``Fp8Tensor`` stands beside ``moe.Q4Tensor``: ``ExpertWeights(Fp8Tensor, Fp8Tensor)``
makes ``routed_experts`` and ``moe_block`` run on 8-bit experts, forward and
grad-input, and ``fp8_linear`` is the product for one weight.  Activations are
quantized in the call.  The weights are frozen: gradients go to the activations,
and to the positions a ``SparseGradStore`` samples.

The reference has no 8-bit format; its frozen weights are 4-bit
(usaf/quantization.py:21-132) or dense.
"""
from __future__ import annotations

import contextlib
import functools
from typing import NamedTuple, Optional, Sequence, Tuple

import torch

from . import _native as N

BLOCK = 128
_ACT = (torch.float16, torch.bfloat16)


def _blocks(n: int) -> int:
    return -(-n // BLOCK)


_HERE = contextlib.nullcontext()


def on(device: torch.device):
    """The device made current for a call's launches (nothing to do where it is)."""
    return _HERE if device.index == torch.cuda.current_device() else torch.cuda.device(device)


@functools.lru_cache(maxsize=4096)
def _linear_ws_bytes(m: int, k: int) -> int:
    return N.load().usaf_hip_fp8_linear_ws_bytes(m, k)


class Fp8Tensor:
    """An HBM-resident weight [R, C] or [E, R, C] in the 8-bit block format.

    q: e4m3 codes (uint8 or float8_e4m3fn), [.., R, 128 * ceil(C / 128)], zeros behind
    column C; s: E8M0 bytes (uint8), [.., ceil(R / 128), ceil(C / 128)], from 7 to 247 as the codec
    writes them.  The tensors are used as they are; a code behind column C that is not zero gives
    wrong products, and a value past bf16's range is infinite in some.
    They are not written to once the weight has been used, and a weight is kept until the
    work that reads it, on whichever streams, has ended."""

    def __init__(self, q: torch.Tensor, s: torch.Tensor, shape: Sequence[int]):
        shape = torch.Size(int(d) for d in shape)
        if len(shape) not in (2, 3) or any(d < 1 for d in shape):
            raise ValueError(f"Fp8Tensor: shape must be [R, C] or [E, R, C] with no empty dimension, got {tuple(shape)}")
        if q.dtype == torch.float8_e4m3fn:
            q = q.view(torch.uint8)
        if q.dtype != torch.uint8 or s.dtype != torch.uint8:
            raise TypeError(f"Fp8Tensor: codes are e4m3 or uint8 and scales uint8 (E8M0), got {q.dtype}, {s.dtype}")
        *lead, rows, cols = shape
        if tuple(q.shape) != (*lead, rows, _blocks(cols) * BLOCK) or tuple(s.shape) != (*lead, _blocks(rows), _blocks(cols)):
            raise ValueError(f"Fp8Tensor: codes {tuple(q.shape)} and scales {tuple(s.shape)} do not fit {tuple(shape)}: "
                             f"need {(*lead, rows, _blocks(cols) * BLOCK)} and {(*lead, _blocks(rows), _blocks(cols))}")
        if not q.is_contiguous() or not s.is_contiguous() or q.device != s.device or q.data_ptr() % 16:
            raise ValueError("Fp8Tensor: codes and scales must be contiguous, on one device, the codes 16-byte aligned")
        self.q, self.s, self.shape = q, s, shape
        self._t: Optional["Fp8Tensor"] = None

    @classmethod
    def quantize(cls, tensor: torch.Tensor, device=None) -> "Fp8Tensor":
        """From a float weight [R, C] or [E, R, C] (copied to the GPU first where it is on the CPU)."""
        if tensor.dim() not in (2, 3) or tensor.numel() == 0:
            raise ValueError(f"Fp8Tensor.quantize: need a non-empty [R, C] or [E, R, C] tensor, got {tuple(tensor.shape)}")
        N.refuse_followed("Fp8Tensor.quantize", tensor)
        dev = torch.device(device) if device is not None else (tensor.device if tensor.is_cuda else N.default_device())
        if dev.index is None:
            dev = torch.device(dev.type, torch.cuda.current_device())
        w = tensor.detach()
        if w.dtype not in (torch.float32, torch.float16, torch.bfloat16):
            w = w.float()
        w = N.on_device(w, dev)
        *lead, rows, cols = w.shape
        q = torch.empty(*lead, rows, _blocks(cols) * BLOCK, dtype=torch.uint8, device=dev)
        s = torch.empty(*lead, _blocks(rows), _blocks(cols), dtype=torch.uint8, device=dev)
        with on(dev):
            N.call("usaf_hip_fp8_quantize_weight", w.data_ptr(), N.dtype_code(w.dtype), lead[0] if lead else 1, rows, cols,
                   q.data_ptr(), s.data_ptr(), N.stream_ptr(dev))
        return cls(q, s, w.shape)

    def dequantize(self, out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The values, exact in fp32 and bf16 and rounded in fp16, which lacks the smallest."""
        N.refuse_followed("Fp8Tensor.dequantize")
        out = torch.empty(self.shape, dtype=out_dtype, device=self.device)
        with on(self.device):
            N.call("usaf_hip_fp8_dequantize", self.q.data_ptr(), self.s.data_ptr(), *self._erc(), out.data_ptr(),
                   N.dtype_code(out_dtype), N.stream_ptr(self.device))
        return out

    def transposed(self) -> "Fp8Tensor":
        """The transpose (of each matrix), which the grad-input product reads: exact, built
        at the first call (not in a stream capture) and kept (as many bytes again)."""
        if self._t is None:
            N.refuse_capture("Fp8Tensor.transposed: the first call")
            *lead, rows, cols = self.shape
            q = torch.empty(*lead, cols, _blocks(rows) * BLOCK, dtype=torch.uint8, device=self.device)
            s = torch.empty(*lead, _blocks(cols), _blocks(rows), dtype=torch.uint8, device=self.device)
            with on(self.device):
                N.call("usaf_hip_fp8_transpose", self.q.data_ptr(), self.s.data_ptr(), *self._erc(), q.data_ptr(),
                       s.data_ptr(), N.stream_ptr(self.device))
            torch.cuda.current_stream(self.device).synchronize()  # any stream may read it from here on
            self._t = Fp8Tensor(q, s, (*lead, cols, rows))
        return self._t

    def _erc(self) -> Tuple[int, int, int]:
        return (1, *self.shape) if len(self.shape) == 2 else tuple(self.shape)

    @property
    def device(self) -> torch.device:
        return self.q.device

    def numel(self) -> int:
        return self.shape.numel()

    def nbytes(self) -> int:
        return self.q.numel() + self.s.numel()


class Rows(NamedTuple):
    """Quantized activation rows: codes [rows, 128 * ceil(cols / 128)], scale bytes, columns."""
    q: torch.Tensor
    s: torch.Tensor
    cols: int


def empty_rows(rows: int, cols: int, device: torch.device) -> Rows:
    q = torch.empty(rows, _blocks(cols) * BLOCK, dtype=torch.uint8, device=device)
    return Rows(q, torch.empty(rows, -(-_blocks(cols) // 4) * 4, dtype=torch.uint8, device=device), cols)


def quantize_rows(x: torch.Tensor, n_rows: Optional[torch.Tensor] = None) -> Rows:
    """Rows of fp16 / bf16 activations [M, K] in blocks of 128 along the row.  n_rows:
    optional int32 device value; rows from there on are left undefined."""
    if x.dim() != 2 or x.dtype not in _ACT:
        raise TypeError(f"quantize_rows: need fp16 or bf16 rows [M, K], got {x.dtype} {tuple(x.shape)}")
    N.refuse_followed("quantize_rows", x)
    return rows_of(x, n_rows)


def rows_of(x: torch.Tensor, n_rows: Optional[torch.Tensor] = None) -> Rows:
    """quantize_rows inside an autograd function, which a trace records as a whole."""
    if x.stride(1) != 1 or x.stride(0) < x.shape[1]:
        x = x.contiguous()
    rows = empty_rows(x.shape[0], x.shape[1], x.device)
    with on(x.device):
        N.call("usaf_hip_fp8_quantize_rows", x.data_ptr(), N.dtype_code(x.dtype), x.shape[0], x.shape[1],
               max(x.stride(0), x.shape[1]), N.ptr(n_rows), rows.q.data_ptr(), rows.s.data_ptr(), N.stream_ptr(x.device))
    return rows


class Fp8LinearFn(torch.autograd.Function):
    """y = Q(x) W^T; dx = Q(dy) W."""

    @staticmethod
    def forward(ctx, x: torch.Tensor, w: Fp8Tensor):
        ctx.w, ctx.dtype = w, x.dtype
        return _linear(x, w)

    @staticmethod
    def backward(ctx, dy: torch.Tensor):
        if torch.is_grad_enabled():
            raise RuntimeError("fp8_linear has no second derivative (create_graph=True)")
        N.refuse_capture("fp8_linear's backward")
        return _linear(dy if dy.dtype == ctx.dtype else dy.to(ctx.dtype), ctx.w.transposed()), None


def _linear(x: torch.Tensor, w: Fp8Tensor) -> torch.Tensor:
    n, k = w.shape
    dev = x.device
    rows = x if x.dim() == 2 else x.reshape(-1, k) if x.numel() else x.new_empty(0, k)
    m = rows.shape[0]
    if rows.stride(1) != 1 or rows.stride(0) < k:
        rows = rows.contiguous()
    out = torch.empty(m, n, dtype=x.dtype, device=dev)
    if m:
        need = _linear_ws_bytes(m, k)
        with on(dev):
            ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
            N.call("usaf_hip_fp8_linear", rows.data_ptr(), N.dtype_code(x.dtype), m, k, max(rows.stride(0), k),
                   w.q.data_ptr(), w.s.data_ptr(), n, out.data_ptr(), N.ptr(ws), need, N.stream_ptr(dev))
    return out if x.dim() == 2 else out.view(*x.shape[:-1], n)


def fp8_linear(x: torch.Tensor, w: Fp8Tensor) -> torch.Tensor:
    """F.linear with an 8-bit block-scaled weight: x [..., K] fp16 / bf16, w [N, K] ->
    [..., N] in x's dtype.  Differentiable in x (the weight is frozen); the first backward
    builds ``w.transposed()``.  A value of x that is not finite makes its output row NaN.
    A stream capture takes the call without a gradient only, as the graph of a training step
    is switched off (graphs.py).  There is no forward-mode derivative; torch.jit.trace records
    the call.

    Up to 32 rows with rows * K (K in whole blocks) <= 16,384 are summed in fp32.  More rows take the
    8-bit matrix instruction, which drops what lies below about 2^-13 of the largest of the 64
    products that it sums at a time: so a row's result may differ in its last bits with the number of
    rows in the call.  On normal data that is 1.5e-5 of a result (rms): the rms distance to the exact
    product is 2.08e-4 in fp16 and 1.66e-3 in bf16, as by rounding to them alone.  With a column of x 100
    times the others in every 128 it is 2.19e-4 in fp16 (rounding alone 2.07e-4) and 1.66e-3 in bf16.
    A result that remains where much larger products cancel can lose all its digits."""
    if len(w.shape) != 2:
        raise ValueError(f"fp8_linear: need a weight [N, K], got {tuple(w.shape)}")
    if x.dtype not in _ACT:
        raise TypeError(f"fp8_linear: activations must be fp16 or bf16, got {x.dtype}")
    if x.dim() < 1 or x.shape[-1] != w.shape[1]:
        raise ValueError(f"fp8_linear: activations {tuple(x.shape)} do not fit the weight {tuple(w.shape)}")
    if x.device != w.device or not x.is_cuda:
        raise ValueError(f"fp8_linear: activations on {x.device}, weight on {w.device}: both on one GPU")
    if torch.is_grad_enabled() and x.requires_grad:
        N.refuse_capture("fp8_linear of activations that want a gradient")
        return Fp8LinearFn.apply(x, w)
    # (the function's own call takes 2 us of the host's time, beside 7 of a small product's launch)
    return Fp8LinearFn.apply(x, w) if N.followed(x) else _linear(x, w)


# ---------------------------------------------------------------------------
# the routed experts (moe.RoutedExpertsFn)
# ---------------------------------------------------------------------------

# The experts' products whose results are quantized again (gate and up, the gated activation's
# gradient) take the 16-bit matrix instruction.  The 8-bit one is off by 1.5e-5 of a result, which
# neither 16-bit type shows; but values that fall to the other side of a code's border by
# it (a step of up to 2^-3) put an error of about sqrt(1.5e-5 * 2^-4) = 1e-3 into the layer's output, and
# more into its gradients: 1.4 to 1.9 times bf16's own rounding in all, six times fp16's.  The
# two last products, whose results are only rounded, take the 8-bit one.


def experts_forward(x: Rows, ew, b, gu: Optional[torch.Tensor], act: Optional[torch.Tensor], dtype: torch.dtype) -> torch.Tensor:
    """y of the slots of bucketing b from the quantized hidden states, for 8-bit experts ew, with the steps before it in
    gu and act (None: not kept). Each step's output is rounded to dtype, the activations', as on the
    layer's other kernels."""
    S, E, H, I, dev, lib = b.n_slots, ew.E, ew.H, ew.I, x.q.device, N.load()
    with on(dev):
        if gu is None and (act is not None or not lib.usaf_hip_fp8_gate_up_ok(S, E, I, H)):
            gu = torch.empty(S, 2 * I, dtype=dtype, device=dev)
        y = torch.empty(S, H, dtype=dtype, device=dev)
        ws = torch.empty(lib.usaf_hip_fp8_experts_fwd_ws_bytes(S, I), dtype=torch.uint8, device=dev)
        N.call("usaf_hip_fp8_experts_fwd", x.q.data_ptr(), x.s.data_ptr(), x.q.shape[0], b.token_idx.data_ptr(),
               b.offsets.data_ptr(), S, E, H, I, N.dtype_code(dtype), ew.gate_up.q.data_ptr(), ew.gate_up.s.data_ptr(),
               ew.down.q.data_ptr(), ew.down.s.data_ptr(), N.ptr(gu), N.ptr(act), y.data_ptr(), ws.data_ptr(), ws.numel(),
               N.stream_ptr(dev))
    return y


def experts_bwd(dout: torch.Tensor, y: torch.Tensor, gu: torch.Tensor, ew, b, dcur: Optional[torch.Tensor],
                dgu: Optional[torch.Tensor], dweights: torch.Tensor) -> torch.Tensor:
    """The slots' gradient of the hidden states; that of the routing weights goes to dweights (zeros before), those of
    the experts' outputs and of gu to dcur and dgu (None: not kept)."""
    S, H = y.shape
    E, I, dev = ew.E, ew.I, y.device
    down, gate_up = ew.down.transposed(), ew.gate_up.transposed()
    dx_slots = torch.empty(S, H, dtype=y.dtype, device=dev)
    ws = torch.empty(N.load().usaf_hip_fp8_experts_bwd_ws_bytes(S, H, I), dtype=torch.uint8, device=dev)
    with on(dev):
        N.call("usaf_hip_fp8_experts_bwd", dout.data_ptr(), y.data_ptr(), gu.data_ptr(), b.token_idx.data_ptr(),
               b.slot_w.data_ptr(), b.offsets.data_ptr(), S, E, H, I, N.dtype_code(y.dtype), down.q.data_ptr(),
               down.s.data_ptr(), gate_up.q.data_ptr(), gate_up.s.data_ptr(), N.ptr(dcur), N.ptr(dgu), dx_slots.data_ptr(),
               dweights.data_ptr(), ws.data_ptr(), ws.numel(), N.stream_ptr(dev))
    return dx_slots
