"""How the framework's other calls meet a model in 8 bits, without a GPU."""

from __future__ import annotations

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
