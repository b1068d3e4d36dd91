"""ModelRunner and LLMEngine with drafted tokens: errors, blocks, drafts and the steps they save."""

from __future__ import annotations

import random

import pytest
import torch

from tests.test_speculative_gpu import dense_logits

pytestmark = pytest.mark.gpu

VOCAB = 101


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA GPU")
    return torch.device("cuda", 0)


def make_model(dev, dtype=torch.float16, **extra):
    from mini_inference_b200.model import Qwen2Config, Qwen2Model, init_random

    cfg = Qwen2Config(vocab_size=VOCAB, hidden_size=256, intermediate_size=320, num_layers=2, num_heads=6, num_kv_heads=2, head_dim=64,
                      max_position_embeddings=512, rope_theta=1e4, **extra)
    return Qwen2Model(cfg, init_random(cfg, seed=3, std=0.08, dtype=dtype, device=dev, unit_norms=True))


def make_engine(model, **config):
    from mini_inference_b200.engine import EngineConfig, LLMEngine

    eos = config.pop("eos", ())
    settings = dict(max_num_seqs=4, max_model_len=160, max_num_batched_tokens=256, kv_cache_tokens=640) | config
    return LLMEngine(model, EngineConfig(**settings), eos_token_ids=eos)


def check_greedy(model, seqs):
    """Every token within float16 rounding of the dense float64 forward's best logit (the engine tests' rule)."""
    for s in seqs:
        rows = dense_logits(model, model.cfg, s.token_ids)[s.prompt_len - 1:-1]
        best = rows.amax(-1)
        got = rows.gather(1, torch.tensor(s.output_token_ids, device=model.device)[:, None])[:, 0]
        assert (got >= best - 0.02 * best.abs().clamp(min=1.0)).all(), (best - got).max()


def prompts_of(seed=4):
    rng = random.Random(seed)
    phrase = [rng.randrange(VOCAB) for _ in range(9)]
    return [phrase * 3 + phrase[:4], [rng.randrange(VOCAB) for _ in range(31)], phrase[:5] * 2, phrase + [3] * 12]


def test_an_error_of_the_lm_head_is_raised(dev):
    """verify_tokens reads the LM head's status word, as a decode step does."""
    engine = make_engine(make_model(dev), speculative_tokens=4)
    slot = engine.cache.allocate(8)
    engine.runner.prefill_tokens([slot], [[1, 2, 3, 4]])
    assert engine.runner.verify_tokens([slot], [([5], [-1])])
    engine.runner.head.status.fill_(9)  # what a timed-out wait leaves
    with pytest.raises(RuntimeError, match="timed out"):
        engine.runner.verify_tokens([slot], [([6], [-1])])
    assert engine.runner.verify_tokens([slot], [([7], [-1])])  # cleared


def test_drafts_take_no_block_that_a_decode_step_needs(dev):
    """A pool in which plain decoding preempts nothing: nor does drafting, and the tokens are still greedy choices.

    Four sequences end at 71, 71, 50 and 61 tokens, 18 blocks of 16 in all, as many as there are.
    """
    from mini_inference_b200.engine import SamplingParams

    model, prompts = make_model(dev), prompts_of()
    params = SamplingParams(max_tokens=40, ignore_eos=True)
    for speculative in (0, 40):
        engine = make_engine(model, max_model_len=80, kv_cache_tokens=18 * 16, speculative_tokens=speculative)
        for p in prompts:
            engine.add_request(p, params)
        while engine.has_unfinished_requests():
            engine.step()
            for s in engine.scheduler.running:
                assert len(engine.cache.block_tables[s.slot]) <= engine.cache.blocks_for(s.num_tokens)
        engine.check_device_errors()
        assert engine.scheduler.num_preemptions == 0
        assert engine.cache.num_free_blocks == 18
        check_greedy(model, engine.sequences.values())


def test_a_tree_gives_back_what_its_path_left_unused(dev):
    from mini_inference_b200 import PagedKVCache

    cache = PagedKVCache(1, 2, 64, num_blocks=12, block_size=16, max_seqs=3, max_len=160, dtype=torch.float16, device=dev)
    a, b = cache.allocate(10), cache.allocate(60)  # the second one's spare blocks are its caller's own
    cache.lengths[a], cache.lengths[b] = 10, 15
    ctx = cache.tree_context([a, b], [[-1] + list(range(40)), [-1, 0]])
    assert len(cache.block_tables[a]) == 4 and len(cache.block_tables[b]) == 4
    x = torch.randn(1, 2, 43, 64, device=dev).half()
    ctx.attend(0, x, x, x)
    ids = torch.arange(43, device=dev)
    assert ctx.accept(ids, ids + 1000) == [[1000], [1041]]  # nothing drafted is right
    assert len(cache.block_tables[a]) == 1 and len(cache.block_tables[b]) == 4 and cache.num_free_blocks == 7
    ctx = cache.tree_context([a, b], [[-1] + list(range(40)), [-1, 0]])
    ctx.attend(0, x, x, x)
    assert [len(row) for row in ctx.accept(ids, ids + 1)] == [41, 2]  # all of it is
    assert cache.lengths[a] == 52 and len(cache.block_tables[a]) == 4 and len(cache.block_tables[b]) == 4
    cache.raise_device_errors()


def test_a_step_without_a_draft_is_a_plain_decode(dev):
    """It goes through the captured decode graph: the last token of a request leaves no room for a draft."""
    from mini_inference_b200.engine import SamplingParams

    model = make_model(dev)
    engine = make_engine(model, speculative_tokens=8)
    seqs = engine.generate([[7], [9, 8, 7]], SamplingParams(max_tokens=2, ignore_eos=True))
    assert engine.runner.graphs.replays == 1 and len(engine.step_stats) == 2
    check_greedy(model, seqs)
    # Steps with and without drafts in turn, on one cache.
    engine = make_engine(model, speculative_tokens=3)
    seqs = engine.generate(prompts_of(6), SamplingParams(max_tokens=50, ignore_eos=True))
    assert 0 < engine.runner.graphs.replays < len(engine.step_stats)
    check_greedy(model, seqs)
