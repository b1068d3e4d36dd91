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
