"""A layer's projections in microscaled 4 bits without a GPU: which weights and which activation it
holds for the kinds of MLP that the drafter's module takes."""

from types import SimpleNamespace

import pytest
import torch

from flashmap_amd import ops
from flashmap_amd.draft_step import MXLayer
from flashmap_amd.drafter import FlashMapLayer, drafter_config


@pytest.mark.parametrize("kind,activation", [("gelu", "gelu"), ("swiglu", "swiglu"), ("mlp", "gelu"), (None, "gelu")])
def test_activation_is_the_modules(monkeypatch, kind, activation):
    """The module (flashmap/modeling_flashmap.py:150-170) takes every type but "swiglu" as GELU, and a
    configuration that is a namespace already is used as it is."""
    asked = []
    monkeypatch.setattr(ops, "mx_quantize", lambda x, bits=8, activation=None: asked.append(activation) or (x, bits))
    monkeypatch.setattr(ops, "mx_linear", lambda x, w, bias=None, out=None: x)
    cfg = drafter_config(SimpleNamespace(**vars(drafter_config(hidden_size=64, num_attention_heads=2, cond_dim=8,
                                                               time_embed_dim=8, intermediate_size=96)) | {"mlp_type": kind}))
    layer = FlashMapLayer(cfg)
    held = MXLayer(layer, torch.zeros(192, 64))
    up, down = (layer.mlp.gate_up_proj, layer.mlp.down_proj) if kind == "swiglu" else (layer.mlp.fc1, layer.mlp.fc2)
    assert held.up == (up.weight, 4) and held.down == (down.weight, 4)
    assert held.up_bias is up.bias and held.down_bias is down.bias
    asked.clear()
    held.mlp(torch.zeros(2, 64))
    assert asked == [activation]
