"""Layer settings that no model has are refused when it is built. No GPU needed."""

from __future__ import annotations

import pytest
import torch

from mini_inference_b200.model import Qwen2Config, Qwen2Model, init_random, parameter_shapes


def build(**kw):
    cfg = Qwen2Config(vocab_size=11, hidden_size=64, intermediate_size=64, num_layers=1, num_heads=2, num_kv_heads=1, head_dim=64,
                      max_position_embeddings=32, **kw)
    return Qwen2Model(cfg, init_random(cfg, seed=1, dtype=torch.float16, device="cpu"))


@pytest.mark.parametrize("bad", [dict(rope_sections=(8, 8, 8)), dict(rope_sections=(8, 8, 8, 8)), dict(rope_sections=()),
                                 dict(rope_sections=(40, -8)), dict(num_experts=2, experts_per_token=3),
                                 dict(num_experts=32, experts_per_token=17), dict(num_experts=2, experts_per_token=0)])
def test_refused(bad):
    with pytest.raises(ValueError):
        build(**bad)


def test_parameters():
    cfg = build(qk_norm=True, num_experts=4, expert_intermediate_size=24).cfg
    shapes = dict(parameter_shapes(cfg))
    assert shapes["layers.0.attn.q_norm.weight"] == shapes["layers.0.attn.k_norm.weight"] == (64,)
    assert shapes["layers.0.mlp.router.weight"] == (4, 64)
    assert shapes["layers.0.mlp.experts.gate_up_proj.weight"] == (4, 48, 64)
    assert shapes["layers.0.mlp.experts.down_proj.weight"] == (4, 64, 24)
    assert "layers.0.mlp.down_proj.weight" not in shapes


def test_what_goes_through_which_rotation():
    plain = build()
    assert plain.rotary is None and plain.head_norms == [None] and plain.routers == []
    norms = build(qk_norm=True)
    assert norms.rotary.inv_freq.numel() == 32 and norms.rotary.axes is None and norms.cos is None
    axes = build(rope_sections=(8, 12, 12))
    assert axes.rotary.axes.tolist() == [0] * 8 + [1] * 12 + [2] * 12
    half = build(rope_sections=(6, 5, 5), rope_sections_alternate=True, rotary_dim=32)
    assert half.rotary.axes.tolist() == [0, 1, 2] * 5 + [0]
