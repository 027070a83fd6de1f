"""Drop-in replacements for the reference's patched Qwen3-MoE forwards.

``patch_qwen3moe_for_dml()`` installs, exactly like usaf/qwen3moe_dml.py:89-94,

* ``Qwen3MoeExperts.forward(self, hidden_states [N, H], weights [N, E])`` and
* ``Qwen3MoeSparseMoeBlock.forward(self, hidden_states [B, S, H])``,

but the expert math runs on the routed tokens only, through the fused 4-bit
dequant-GEMM kernels (when the module carries HBM 4-bit tensors in
``module._usaf_q4``, set by ``moe_loader.setup_quantized_streaming``) or the
dense-weight variant of the same kernels (``self.gate_up_proj`` /
``self.down_proj``).  The result equals the reference's dense-masked sum:
non-routed experts contribute exact zeros there.

Grad capture keeps the reference protocol: with
``module._grad_capture = (store, prefix)`` the weight gradients of
``{prefix}.gate_up_proj`` / ``{prefix}.down_proj`` go to ``store`` -- sampled
at the active positions for ``usaf_amd.moe_loader.SparseGradStore``, as dense
per-expert tensors (``store.add(name, ei, g)`` or a dict of fp16 buffers) for
other stores.  The expert weights themselves receive no ``.grad``, as in the
reference (it detaches every per-expert slice).

Decoding: with ``block._usaf_few_tokens = n`` (up to 32) a block's passes of at most
n tokens that want no gradient run as ``few.few_token_block``, router and experts in
three or four launches, where the experts are 4-bit or 8-bit (attached to the experts module, or streamed by
``moe_loader.setup_quantized_streaming``) and carry no trained values.  Such a pass does not call the experts
module: its hooks do not run, and copies of its weights (``expert_cache_bytes``) are not used.
Its numerics (``few.py``) differ from this path's in what is rounded to 16 bits, so it is off by default.
"""
from __future__ import annotations

import torch

from .few import few_token_block, few_token_ok
from .moe import ExpertWeights, RouteTopKFn, routed_experts


def _with_overlays(gate_up, down, overlays) -> ExpertWeights:
    ew = ExpertWeights(gate_up, down)
    # trained values over the 4-bit weights (QuantizedExpertCache.sync_resident)
    for local, ov in (overlays or {}).items():
        ew.overlays[local.replace("_proj", "")] = ov
    return ew


def _expert_weights(module) -> ExpertWeights:
    q4 = getattr(module, "_usaf_q4", None)
    if q4:
        gu, dn = q4.get("gate_up_proj"), q4.get("down_proj")
        if gu is None or dn is None:
            raise RuntimeError("module._usaf_q4 must hold gate_up_proj and down_proj")
        return _with_overlays(gu, dn, getattr(module, "_usaf_q4_overlays", None))
    gu = getattr(module, "gate_up_proj", None)
    dn = getattr(module, "down_proj", None)
    if gu is None or dn is None:
        raise RuntimeError("expert module has no weights: attach 4-bit tensors (module._usaf_q4) or "
                           "dense gate_up_proj/down_proj")
    return ExpertWeights(gu.detach(), dn.detach())


def _slot_cache_of(module, hidden_states: torch.Tensor, weights: torch.Tensor, capture):
    """The per-expert copy cache for this forward, if it may serve it: no
    gradient is wanted, the module carries no trained values (their masters
    change every step; the fused GEMMs read them through overlay tables) and
    the activations are in the copies' dtype."""
    slots = getattr(module, "_usaf_slots", None)
    if slots is None or capture is not None or getattr(module, "_usaf_q4_overlays", None):
        return None
    if torch.is_grad_enabled() and (hidden_states.requires_grad or weights.requires_grad):
        return None
    cache, name = slots
    return slots if hidden_states.dtype == cache.dtype else None


def dml_qwen3_experts_forward(self, hidden_states: torch.Tensor, weights: torch.Tensor) -> torch.Tensor:
    """qwen3moe_dml.py:24-64: [N, H] x routing weights [N, E] -> [N, H]."""
    capture = None
    if torch.is_grad_enabled() and getattr(self, "_grad_capture", None) is not None:
        capture = self._grad_capture
    slots = _slot_cache_of(self, hidden_states, weights, capture)
    if slots is not None:
        cache, name = slots
        return cache.forward(name, hidden_states.contiguous(), weights.to(cache.dtype).contiguous())
    return routed_experts(hidden_states, weights, _expert_weights(self), capture)


def _few_weights(block, hs: torch.Tensor):
    """The experts of a pass that few_token_block takes for this block, or None."""
    limit = getattr(block, "_usaf_few_tokens", 0)
    if not 0 < hs.shape[0] <= limit:
        return None
    experts, router = block.experts, block.gate
    if torch.is_grad_enabled() and (hs.requires_grad or router.weight.requires_grad
                                    or getattr(experts, "_grad_capture", None) is not None):
        return None
    if router.weight.dtype != hs.dtype:
        return None
    q4, overlays = getattr(experts, "_usaf_q4", None), getattr(experts, "_usaf_q4_overlays", None)
    source = getattr(experts, "_usaf_q4_source", None)
    if source is not None:  # a streamed module, whose hooks attach its weights in its own call only
        q4, overlays = source(experts)
    if not q4 or q4.get("gate_up_proj") is None or q4.get("down_proj") is None:
        return None
    ew = _with_overlays(q4["gate_up_proj"], q4["down_proj"], overlays)
    return ew if few_token_ok(hs.shape[0], int(router.top_k), ew) else None


def dml_qwen3_moe_block_forward(self, hidden_states: torch.Tensor) -> torch.Tensor:
    """qwen3moe_dml.py:67-86: router linear, fp32 softmax, >=-threshold top-k
    mask, optional renormalisation, routed experts."""
    batch_size, sequence_length, hidden_dim = hidden_states.shape
    hs = hidden_states.view(-1, hidden_dim)
    router = self.gate
    ew = _few_weights(self, hs)
    if ew is not None:
        out = few_token_block(hs, router.weight, int(router.top_k), bool(getattr(router, "norm_topk_prob", False)), ew)
        return out.view(batch_size, sequence_length, hidden_dim)
    router_logits = torch.nn.functional.linear(hs, router.weight)
    weights = RouteTopKFn.apply(router_logits, int(router.top_k), bool(getattr(router, "norm_topk_prob", False)),
                                hs.dtype)
    final = self.experts(hs, weights)
    return final.view(batch_size, sequence_length, hidden_dim)


def patch_qwen3moe_for_dml():
    """Install the forwards on transformers' Qwen3-MoE classes (all instances)."""
    from transformers.models.qwen3_moe import modeling_qwen3_moe
    modeling_qwen3_moe.Qwen3MoeExperts.forward = dml_qwen3_experts_forward
    modeling_qwen3_moe.Qwen3MoeSparseMoeBlock.forward = dml_qwen3_moe_block_forward
    return modeling_qwen3_moe
