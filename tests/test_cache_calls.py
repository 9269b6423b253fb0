"""Calls of the cached-generation paths that must be refused, or leave things as
they are, without a GPU."""

from __future__ import annotations

import pytest
import torch


def _model():
    from SSA.ssa_decoder import SSADecoder, SSADecoderConfig

    return SSADecoder(SSADecoderConfig(num_layers=1, hidden_size=64, num_attention_heads=1, num_query_groups=1,
                                       kv_channels=64, ffn_hidden_size=64, vocab_size=64))


def test_a_tree_needs_caches():
    """A tree's mask without caches would be the plain causal forward's, unseen."""
    model = _model()
    ids, mask = torch.zeros(2, 4, dtype=torch.long), torch.eye(4, dtype=torch.bool)
    with pytest.raises(ValueError, match="caches"):
        model(ids, tree_mask=mask)
    with pytest.raises(ValueError, match="caches"):
        model(ids, positions=torch.zeros(2, 4, dtype=torch.long), tree_mask=mask)
    layer = model.layers[0]
    x = torch.zeros(4, 2, 64)
    with pytest.raises(ValueError, match="cache"):
        layer.self_attention(x, model.rotary(torch.arange(4)), None, mask)
