"""A whole MoE layer for a few tokens, as decoding calls it.

``few_token_block`` is ``moe.moe_block`` for 1 to 32 tokens without gradients, on
4-bit (``Q4Tensor``) or 8-bit (``Fp8Tensor``) experts: router, top-k, the experts in
use and their weighted sum in three or four launches, with no host read and no state
between calls.  It keeps more digits than the routed path between its steps
(usaf/qwen3moe_dml.py:24-86 rounds each op's output to the activations' dtype):

* the router's logits are not rounded to 16 bits.  Exactly ``top_k`` experts serve
  each token, the lowest-numbered of equal ones (to 44 bits), where the 16-bit rule
  takes all experts that tie at the threshold;
* gate, up, each expert's output and the routing weights stay in fp32; only the
  gated activation, the operand of the second product, is rounded;
* a 4-bit weight is code * scale + zero as a real number, without the codec's fp16
  roundings; with 8-bit experts the activations are not quantized.
"""
from __future__ import annotations

import functools

import torch

from . import _native as N
from .fp8 import on
from .moe import ExpertWeights, Q4Tensor

MAX_TOKENS = 32
MAX_EXPERTS = 256
MAX_TOP_K = 16


@functools.lru_cache(maxsize=1024)
def _ws_bytes(device: int, tokens: int, experts: int, top_k: int, hidden: int, inter: int) -> int:
    """The workspace on a device (its CU count decides the split), which is the current one."""
    return N.load().usaf_hip_moe_few_ws_bytes(tokens, experts, top_k, hidden, inter)


def few_token_ok(tokens: int, top_k: int, experts: ExpertWeights) -> bool:
    """Whether few_token_block takes this many tokens on these experts."""
    gu, dn = experts.gate_up, experts.down
    coded = experts.is_fp8 or (isinstance(gu, Q4Tensor) and isinstance(dn, Q4Tensor) and gu.fused_ok() and dn.fused_ok())
    return (coded and not experts.overlays and 0 <= tokens <= MAX_TOKENS and experts.E <= MAX_EXPERTS
            and 1 <= top_k <= min(MAX_TOP_K, experts.E) and experts.H % 128 == 0 and experts.I % 128 == 0
            and experts.H <= 16384 and experts.I <= 65536)


def few_token_block(hs: torch.Tensor, router_weight: torch.Tensor, top_k: int, norm_topk_prob: bool,
                    experts: ExpertWeights) -> torch.Tensor:
    """hs [..., H] fp16 / bf16 with at most 32 tokens, router_weight [E, H] of the same
    dtype -> the layer's output, shaped as hs.  No gradients: call it under
    ``torch.no_grad()`` or with tensors that need none, nor forward-mode derivatives
    (torch.jit.trace records the call).  Experts that carry trained values
    (overlays), dense experts and more tokens go through ``moe.moe_block``."""
    dt, dev = hs.dtype, hs.device
    if dt not in (torch.float16, torch.bfloat16) or router_weight.dtype != dt:
        raise TypeError(f"few_token_block: activations and router must be fp16 or bf16 alike, got {dt}, {router_weight.dtype}")
    E, H, I = experts.E, experts.H, experts.I
    if hs.dim() < 1 or hs.shape[-1] != H or router_weight.shape != (E, H):
        raise ValueError(f"few_token_block: activations {tuple(hs.shape)}, router {tuple(router_weight.shape)} and experts "
                         f"E={E} H={H} I={I} do not fit")
    tokens = hs.numel() // H
    if tokens > MAX_TOKENS:
        raise ValueError(f"few_token_block: at most {MAX_TOKENS} tokens, got {tokens} (moe.moe_block takes more)")
    if experts.overlays:
        raise NotImplementedError("few_token_block: experts with trained values (overlays) go through moe.moe_block")
    if not few_token_ok(tokens, top_k, experts):
        raise NotImplementedError(
            f"few_token_block: needs 4-bit (group size 128 along whole rows) or 8-bit experts, H <= 16384 and I <= 65536 in "
            f"multiples of 128, at most {MAX_EXPERTS} experts and 1 <= top_k <= {MAX_TOP_K}; got E={E} H={H} I={I} top_k={top_k}")
    gu, dn = experts.gate_up, experts.down
    if not hs.is_cuda or any(d != dev for d in (router_weight.device, gu.device, dn.device)):
        raise ValueError(f"few_token_block: activations on {dev}, router on {router_weight.device}, experts on {gu.device}: "
                         "all on one GPU")
    if torch.is_grad_enabled() and (hs.requires_grad or router_weight.requires_grad):
        raise RuntimeError("few_token_block has no backward: call it under torch.no_grad(), or moe.moe_block")
    layer = FewTokensFn.apply if N.followed(hs, router_weight) else _layer
    return layer(hs, router_weight, top_k, norm_topk_prob, experts)


def _layer(hs: torch.Tensor, router_weight: torch.Tensor, top_k: int, norm_topk_prob: bool,
           experts: ExpertWeights) -> torch.Tensor:
    dt, dev = hs.dtype, hs.device
    E, H, I, gu, dn = experts.E, experts.H, experts.I, experts.gate_up, experts.down
    tokens = hs.numel() // H
    x = _aligned(hs)
    router = _aligned(router_weight)
    out = torch.empty(hs.shape, dtype=dt, device=dev)
    if tokens == 0:
        return out
    with on(dev):
        gu_s, dn_s = (gu.s, dn.s) if experts.is_fp8 else (gu.scale_zero_by_group(), dn.scale_zero_by_group())
        ws = torch.empty(_ws_bytes(dev.index, tokens, E, top_k, H, I), dtype=torch.uint8, device=dev)
        N.call("usaf_hip_moe_few", x.data_ptr(), tokens, H, router.data_ptr(), E, top_k, 1 if norm_topk_prob else 0,
               N.dtype_code(dt), I, 1 if experts.is_fp8 else 0, gu.q.data_ptr(), gu_s.data_ptr(), dn.q.data_ptr(),
               dn_s.data_ptr(), out.data_ptr(), ws.data_ptr(), ws.numel(), N.stream_ptr(dev))
    return out


class FewTokensFn(torch.autograd.Function):
    """The layer as one operation, for a trace to record and forward-mode derivatives to be refused by."""

    @staticmethod
    def forward(ctx, hs: torch.Tensor, router_weight: torch.Tensor, top_k: int, norm_topk_prob: bool,
                experts: ExpertWeights) -> torch.Tensor:
        return _layer(hs, router_weight, top_k, norm_topk_prob, experts)

    @staticmethod
    def backward(ctx, dout: torch.Tensor):
        raise RuntimeError("few_token_block has no backward")


def _aligned(t: torch.Tensor) -> torch.Tensor:
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()
