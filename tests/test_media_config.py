"""What is refused of images and video in prompts before anything runs. No GPU needed."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from mini_inference_b200 import PagedKVCache
from mini_inference_b200.engine import LLMEngine, Media


def cache(**kw):
    return PagedKVCache(1, 1, 64, num_blocks=8, block_size=16, max_seqs=2, max_len=64, dtype=torch.float16, device="cpu", **kw)


def test_no_media_with_prefixes_that_go_by_token_ids():
    """Prompts of the same ids around different images would share the first one's keys."""
    with pytest.raises(ValueError, match="image"):
        cache(max_media=1, enable_prefix_caching=True)
    with pytest.raises(ValueError):
        cache(max_media=-1)
    assert cache(max_media=1).max_media == 1 and cache(enable_prefix_caching=True).enable_prefix_caching


def engine(max_media=2):
    """An engine that queues requests and runs none."""
    e = object.__new__(LLMEngine)
    e.config = SimpleNamespace(max_media=max_media)
    e.model = SimpleNamespace(cfg=SimpleNamespace(rope_sections=(8, 12, 12), hidden_size=64))
    e.scheduler, e.sequences, e._next_id = SimpleNamespace(add=lambda seq: None), {}, 0
    return e


def test_a_prompt_may_be_any_iterable_of_ids():
    e = engine()
    for prompt in ([3, 1, 2], (3, 1, 2), iter([3, 1, 2]), (t for t in [3, 1, 2]), torch.tensor([3, 1, 2]).numpy()):
        assert list(e.sequences[e.add_request(prompt)].prompt_token_ids) == [3, 1, 2]


@pytest.mark.parametrize("bad", [Media(2, 1, 2, 2, 2**31), Media(2, 1, 2, 2, 1.5), Media(2.0, 1, 2, 2), Media(2, 1, 2.0, 2),
                                 Media(2, 1, 2, 2, rows=[[0.0] * 64] * 4)])
def test_media_that_no_step_can_place_are_refused_with_the_request(bad):
    """Else the request is queued and every step raises."""
    e = engine()
    with pytest.raises(ValueError):
        e.add_request(range(10), media=[bad])
    assert not e.sequences
    e.add_request(range(10), media=[Media(2, 1, 2, 2, 2**31 - 1, torch.zeros(4, 64))])


def test_spans_are_whole_numbers():
    c = cache(max_media=1)
    slot = c.allocate(20)
    with pytest.raises(TypeError):
        c.set_media(slot, [(2.7, 1, 2, 2, 1)])
    c.set_media(slot, [(torch.tensor(2), 1, 2, 2, 1)])
    assert c._media[slot] == ((2, 1, 2, 2, 1),)
