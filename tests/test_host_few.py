"""The decoding switch of patched blocks on streamed models: which passes take the few-token layer.  No GPU work."""
from types import SimpleNamespace

import pytest
import torch
from torch import nn

from usaf_amd import fp8, moe_loader
from usaf_amd import qwen3moe_dml as Q
from usaf_amd.moe import Q4Tensor

E, H, I, K = 4, 128, 128, 2
NAME = "mlp.experts"


def _q4(*shape):
    n = shape[0] * shape[1] * shape[2] // 128
    return Q4Tensor(torch.zeros(n, 64, dtype=torch.int8), torch.ones(n, dtype=torch.float16), torch.zeros(n, dtype=torch.float16),
                    torch.Size(shape))


def _fp8(*shape):
    return fp8.Fp8Tensor(torch.zeros(*shape, dtype=torch.uint8), torch.zeros(shape[0], shape[1] // 128, shape[2] // 128,
                                                                            dtype=torch.uint8), shape)


class Experts(nn.Module):
    forward = Q.dml_qwen3_experts_forward


class Block(nn.Module):
    forward = Q.dml_qwen3_moe_block_forward

    def __init__(self):
        super().__init__()
        self.experts = Experts()
        self.gate = SimpleNamespace(weight=torch.ones(E, H, dtype=torch.bfloat16), top_k=K, norm_topk_prob=True)


class Store(moe_loader.QuantizedExpertCache):
    """The loader's store without a GPU."""

    def __init__(self, entries, device, **_):
        self._q_dict, self._device = dict(entries), torch.device("cpu")
        self.overlays, self.fused_overlays, self._fused_fresh = {}, {}, set()
        self.fused_dtype = self.slot_cache = None
        self._prefetched = {}
        self._build_index()


@pytest.fixture
def streamed(monkeypatch):
    """A streamed model of one block; its calls, and the weights that each read, go to `took`."""
    took = []

    def few(hs, router, k, norm, ew):
        took.append(("few", ew))
        return torch.zeros_like(hs)

    def routed(hs, weights, ew, capture=None):
        took.append(("routed", ew))
        return torch.zeros_like(hs)

    monkeypatch.setattr(moe_loader, "QuantizedExpertCache", Store)
    monkeypatch.setattr(Q, "few_token_block", few)
    monkeypatch.setattr(Q, "routed_experts", routed)
    monkeypatch.setattr(Q, "RouteTopKFn", SimpleNamespace(apply=lambda logits, k, norm, dtype: logits.to(dtype)))
    model = nn.Module()
    model.mlp = Block()
    moe_loader.setup_quantized_streaming(model, {f"{NAME}.gate_up_proj": _q4(E, 2 * I, H), f"{NAME}.down_proj": _q4(E, H, I)},
                                         torch.device("cpu"), expert_pattern="*mlp.experts", verbose=False)
    return model, model._quantized_cache, took


def _pass(model, tokens=3):
    with torch.no_grad():
        return model.mlp(torch.ones(1, tokens, H, dtype=torch.bfloat16))


def test_a_streamed_block_takes_its_few_token_passes_there(streamed):
    model, cache, took = streamed
    _pass(model)
    model.mlp._usaf_few_tokens = 8
    _pass(model)
    _pass(model, 9)
    model.mlp(torch.ones(1, 3, H, dtype=torch.bfloat16, requires_grad=True))
    assert [t for t, _ in took] == ["routed", "few", "routed", "routed"]
    assert all(ew.gate_up is cache._q_dict[f"{NAME}.gate_up_proj"] and not ew.overlays for _, ew in took)
    assert model.mlp.experts._usaf_q4 is None


def test_trained_values_keep_the_routed_path(streamed):
    model, cache, took = streamed
    model.mlp._usaf_few_tokens = 8
    _pass(model)
    overlay = object()
    cache.fused_overlays[f"{NAME}.down_proj"] = SimpleNamespace(ov=overlay, dense=None)
    _pass(model)
    cache.fused_overlays[f"{NAME}.down_proj"] = SimpleNamespace(ov=None, dense=torch.zeros(E, H, I, dtype=torch.bfloat16))
    _pass(model)
    assert [t for t, _ in took] == ["few", "routed", "routed"]
    assert took[1][1].overlays == {"down": overlay} and isinstance(took[2][1].down, torch.Tensor)


def test_a_pass_that_ended_in_an_error_leaves_no_old_weights(streamed):
    model, cache, took = streamed
    model.mlp._usaf_few_tokens = 8
    model.mlp.experts._usaf_q4 = {"gate_up_proj": _q4(E, 2 * I, H), "down_proj": _q4(E, H, I)}  # the post-hook did not run
    _pass(model)
    assert took[-1][1].gate_up is cache._q_dict[f"{NAME}.gate_up_proj"]


def test_a_layer_whose_weights_are_freed(streamed):
    model, cache, _ = streamed
    model.mlp._usaf_few_tokens = 8
    cache._q_dict.clear()
    cache._expert_to_params.clear()
    with pytest.raises(RuntimeError, match="no weights"):
        _pass(model)


def test_attached_8_bit_weights_stay(streamed):
    """8-bit tensors that the user attaches to a streamed module serve every pass of it, its 4-bit ones none."""
    model, cache, took = streamed
    mine = {"gate_up_proj": _fp8(E, 2 * I, H), "down_proj": _fp8(E, H, I)}
    model.mlp.experts._usaf_q4 = mine
    cache.slot_cache = SimpleNamespace(layers={NAME: None}, dtype=torch.bfloat16)
    _pass(model)
    model.mlp._usaf_few_tokens = 8
    _pass(model)
    _pass(model, 9)
    assert [t for t, _ in took] == ["routed", "few", "routed"]
    assert all(ew.gate_up is mine["gate_up_proj"] and ew.down is mine["down_proj"] for _, ew in took)
    assert model.mlp.experts._usaf_q4 is mine
    for ov, dense in ((object(), None), (None, torch.zeros(E, H, I, dtype=torch.bfloat16))):  # never left out in silence
        cache.fused_overlays[f"{NAME}.down_proj"] = SimpleNamespace(ov=ov, dense=dense)
        for tokens in (3, 9):
            with pytest.raises(NotImplementedError, match="trained values"):
                _pass(model, tokens)
    model.mlp.experts._usaf_q4 = None  # back to the streamed ones
    cache.fused_overlays.clear()
    cache.slot_cache = None
    _pass(model)
    assert took[-1][0] == "few" and took[-1][1].gate_up is cache._q_dict[f"{NAME}.gate_up_proj"]
