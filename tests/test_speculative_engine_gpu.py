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


def true_drafts(engine, streams, wrong_every=0):
    """A drafter that knows each request's stream; with `wrong_every` the draft's last token is wrong now and then."""
    calls = [0]

    def draft(seqs, counts, longest=3):
        rows = []
        for s, c in zip(seqs, counts):
            calls[0] += 1
            n = len(s.output_token_ids)
            row = list(streams[s.seq_id][n:n + max(0, c)])
            if wrong_every and row and calls[0] % wrong_every == 0:
                row[-1] = (row[-1] + 1) % VOCAB
            rows.append(row)
        return rows

    engine.scheduler.draft = draft


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_right_drafts_save_steps(dev, dtype):
    """Drafts of 7 tokens, one in three wrong at its end: the same tokens in a fifth of the steps."""
    from mini_inference_b200.engine import SamplingParams

    model, params = make_model(dev, dtype), SamplingParams(max_tokens=40, ignore_eos=True)
    plain = [s.output_token_ids for s in make_engine(model).generate(prompts_of(), params)]
    engine = make_engine(model, speculative_tokens=7)
    true_drafts(engine, plain, wrong_every=3)
    seqs = engine.generate(prompts_of(), params)
    if dtype == torch.float16:
        check_greedy(model, seqs)
    same = 0
    for s, want in zip(seqs, plain):
        # Near-ties may part the streams (other batch shapes round differently); from there the drafts are wrong.
        k = next((i for i, (a, b) in enumerate(zip(s.output_token_ids, want)) if a != b), 40)
        same += k
        if k < 40:
            row = dense_logits(model, model.cfg, s.token_ids[:s.prompt_len + k])[-1]
            # bfloat16's half step is eight times float16's
            tol = (0.02 if dtype == torch.float16 else 0.16) * max(1.0, float(row.max()))
            assert row[s.output_token_ids[k]] >= row.max() - tol and row[want[k]] >= row.max() - tol
    assert same >= 80
    if same == 160:
        assert len(engine.step_stats) <= 8


def test_an_end_token_inside_an_accepted_path(dev):
    """What comes after it is dropped, its request ends there, the others go on, and every block comes back."""
    from mini_inference_b200.engine import SamplingParams

    model = make_model(dev)
    params = SamplingParams(max_tokens=40, ignore_eos=True)
    plain = [s.output_token_ids for s in make_engine(model).generate(prompts_of(), params)]
    # A token first met in the middle of the first stream: between two ends of drafts of 9.
    eos = next(t for i, t in enumerate(plain[0]) if i >= 4 and i % 10 in (3, 4, 5) and t not in plain[0][:i])
    want = [row[:row.index(eos) + 1] if eos in row else row for row in plain]
    engine = make_engine(model, speculative_tokens=9, eos=[eos])
    true_drafts(engine, plain)
    seqs = engine.generate(prompts_of(), SamplingParams(max_tokens=40))
    assert [s.output_token_ids for s in seqs] == want
    assert [s.finish_reason.value for s in seqs] == ["eos" if row[-1] == eos else "length" for row in want]
    assert engine.cache.num_free_blocks == 40 and engine.cache.num_free_slots == 4
    assert sum(len(r) for r in want) == sum(len(s.output_token_ids) for s in seqs)


@pytest.mark.parametrize("chunked", [False, True])
def test_preemption_chunks_and_prefixes_beside_drafts(dev, chunked):
    """A pool too small for all, prompts in chunks (one of which leaves a single token), shared prefixes."""
    from mini_inference_b200.engine import SamplingParams

    model = make_model(dev)
    rng = random.Random(8)
    phrase = [rng.randrange(VOCAB) for _ in range(17)]
    prompts = [phrase + [rng.randrange(VOCAB) for _ in range(rng.randint(1, 20))] for _ in range(7)] + [phrase * 2 + [5], [3]]
    engine = make_engine(model, max_num_seqs=5, max_model_len=96, kv_cache_tokens=192, speculative_tokens=6, enable_prefix_caching=True,
                         chunked_prefill=chunked, max_num_batched_tokens=34 if chunked else 256)
    seqs = engine.generate(prompts, SamplingParams(max_tokens=30, ignore_eos=True))
    assert engine.scheduler.num_preemptions > 0 and engine.cache.prefix_hit_tokens > 0
    assert all(len(s.output_token_ids) == 30 for s in seqs)
    assert engine.cache.num_free_blocks == 12
    check_greedy(model, seqs)


def test_caches_of_more_sequences_than_a_tree_step_takes(dev):
    """1,024 trees at a time (as many as a decode step takes), whatever the cache holds."""
    from mini_inference_b200 import PagedKVCache

    cache = PagedKVCache(1, 2, 64, num_blocks=1100, block_size=16, max_seqs=1100, max_len=32, dtype=torch.float16, device=dev)
    slots = [cache.allocate(2) for _ in range(1025)]
    with pytest.raises(ValueError, match="1024"):
        cache.tree_context(slots, [[-1]] * 1025)
    ctx = cache.tree_context(slots[1:], [[-1]] * 1024)
    x = torch.randn(1, 2, 1024, 64, device=dev).half()
    assert torch.equal(ctx.attend(0, x, x, x), x)  # one key each: its value
    ids = torch.arange(1024, device=dev)
    assert ctx.accept(ids, ids + 7) == [[i + 7] for i in range(1024)]
    cache.raise_device_errors()


def test_a_refused_tree_context_takes_no_block(dev):
    """The first sequence's tree fits, the second's does not (no blocks, or none for its copy of a shared one)."""
    from mini_inference_b200 import PagedKVCache

    chain = [-1] + list(range(40))
    for fork in (False, True):
        cache = PagedKVCache(1, 2, 64, num_blocks=6 if fork else 5, block_size=16, max_seqs=4, max_len=80, dtype=torch.float16, device=dev,
                             enable_copy_on_write=fork)
        a, b = cache.allocate(10), cache.allocate(10)
        cache.lengths[a] = cache.lengths[b] = 10
        c = cache.fork(b) if fork else b
        before = cache._bm.state()
        with pytest.raises(RuntimeError if fork else ValueError):
            cache.tree_context([a, c], [chain, [-1] + list(range(21)) if fork else chain])  # 32 tokens: two blocks, and the copy
        after = cache._bm.state()
        assert {s: len(t) for s, t in after["block_tables"].items()} == {s: len(t) for s, t in before["block_tables"].items()}
        assert sorted(after["free_blocks"]) == sorted(before["free_blocks"]) and after["lengths"] == before["lengths"]


@pytest.mark.parametrize("tree", [False, True])
def test_a_copy_on_write_that_runs_out_keeps_what_it_exchanged(dev, tree):
    """Two forks and one free block: the step is refused, and the first fork's own block has the shared one's rows."""
    from mini_inference_b200 import PagedKVCache

    cache = PagedKVCache(1, 2, 64, num_blocks=3, block_size=16, max_seqs=4, max_len=16, dtype=torch.float16, device=dev,
                         enable_copy_on_write=True)
    a, b = cache.allocate(10), cache.allocate(10)
    cache.lengths[a] = cache.lengths[b] = 10
    cache.k.normal_()
    cache.v.normal_()
    c, d = cache.fork(a), cache.fork(b)
    with pytest.raises(RuntimeError, match="not enough free"):
        cache.tree_context([c, d], [[-1], [-1]]) if tree else cache.decode_context([c, d])
    mine, shared = cache.block_tables[c][0], cache.block_tables[a][0]
    assert mine != shared
    assert torch.equal(cache.k[:, mine], cache.k[:, shared]) and torch.equal(cache.v[:, mine], cache.v[:, shared])
