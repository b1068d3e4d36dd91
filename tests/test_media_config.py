"""What is refused of images and video in prompts before anything runs. No GPU needed."""

from __future__ import annotations

import pytest
import torch

from mini_inference_b200 import PagedKVCache


def cache(**kw):
    return PagedKVCache(1, 1, 64, num_blocks=8, block_size=16, max_seqs=2, max_len=64, dtype=torch.float16, device="cpu", **kw)


def test_no_media_with_prefixes_that_go_by_token_ids():
    """Prompts of the same ids around different images would share the first one's keys."""
    with pytest.raises(ValueError, match="image"):
        cache(max_media=1, enable_prefix_caching=True)
    with pytest.raises(ValueError):
        cache(max_media=-1)
    assert cache(max_media=1).max_media == 1 and cache(enable_prefix_caching=True).enable_prefix_caching
