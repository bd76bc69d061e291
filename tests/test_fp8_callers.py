"""How the framework's other calls meet a model in 8 bits, without a GPU."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from pagedcore_amd import decoder as dec


def _eight_bits(layers: int = 1) -> dec.TinyLlamaWeights:
    """A model whose layers are Fp8LayerWeights of placeholder tensors."""
    weights = dec.random_weights(device="cpu", layers=1, vocab=8, intermediate=16)
    some = torch.zeros((1, 16), dtype=torch.float16)
    rows = dec.Fp8Rows(some, some)
    norm = weights.layers[0].input_norm
    layer = dec.Fp8LayerWeights(norm, rows, rows, norm, rows, rows)
    return dec.TinyLlamaWeights(weights.embedding, (layer,) * layers, weights.final_norm, weights.lm_head)


def test_pack_weights_refuses_a_model_in_8_bits():
    """Its projections are stacked already: quantize_weights's refusal, no AttributeError."""
    with pytest.raises(ValueError, match="already in 8 bits"):
        dec.pack_weights(_eight_bits())


def test_quantize_weights_takes_any_layer_of_the_same_fields(monkeypatch):
    """As the fp16 model does (a caller's own record of the reference's fields): only layers in 8 bits are refused."""
    monkeypatch.setattr(dec, "_quantized", lambda rows: dec.Fp8Rows(rows, rows))
    weights = dec.random_weights(device="cpu", layers=1, vocab=8, intermediate=16)
    own = SimpleNamespace(**vars(weights.layers[0]))
    on_gpu = SimpleNamespace(is_cuda=True)  # the rounding above is the host's
    layer = dec.quantize_weights(dec.TinyLlamaWeights(on_gpu, (own,), weights.final_norm, weights.lm_head)).layers[0]
    assert torch.equal(layer.qkv.values, torch.cat((own.q_proj, own.k_proj, own.v_proj)))
    assert torch.equal(layer.gate_up.values, torch.cat((own.gate_proj, own.up_proj)))
    assert layer.o_proj.values is own.o_proj and layer.down_proj.values is own.down_proj
    eight = dec.TinyLlamaWeights(on_gpu, (layer,), weights.final_norm, weights.lm_head)
    with pytest.raises(ValueError, match="already in 8 bits"):
        dec.quantize_weights(eight)
