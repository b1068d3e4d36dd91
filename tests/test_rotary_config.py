"""Rotary settings of a model that no rotation has are refused when it is built. No GPU needed."""

from __future__ import annotations

import pytest
import torch

from mini_inference_b200.model import Qwen2Config, Qwen2Model, init_random


def build(**kw):
    cfg = Qwen2Config(vocab_size=11, hidden_size=64, intermediate_size=64, num_layers=1, num_heads=2, num_kv_heads=1, head_dim=64,
                      max_position_embeddings=32, **kw)
    return Qwen2Model(cfg, init_random(cfg, seed=1, dtype=torch.float16, device="cpu"))


@pytest.mark.parametrize("rotary_dim", [0, -2, 33, 66, 128])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_dim(rotary_dim, interleaved):
    with pytest.raises(ValueError):
        build(rotary_dim=rotary_dim, rope_interleaved=interleaved)


def test_what_goes_through_which_rotation():
    from mini_inference_b200 import ops

    assert build().rotary is None and build(rotary_dim=64).rotary is None
    part = build(rotary_dim=32)
    assert part.rotary.inv_freq.numel() == 16 and part.cos is None
    assert build(rope_interleaved=True).rotary.inv_freq.numel() == 32
    scaled = build(rope_scaling=ops.RopeScaling("linear", 2.0))
    assert scaled.rotary.inv_freq.numel() == 32 and scaled.cos.shape == (32, 64)
