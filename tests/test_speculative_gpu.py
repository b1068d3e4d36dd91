"""Speculative decoding on the GPU: the operators in a row, as a step uses them.

* Trees through ``TreeContext`` on the engine tests' model, whose greedy streams are far from
  ties (tests/test_engine_gpu.py holds them to a dense float64 oracle): every token that a
  verified tree emits must be the stream's own next one, whatever was drafted.
* ``LLMEngine`` with drafted tokens against the dense float64 forward of the same weights, with
  each rotary layout.
* A whole step on device state, eager and as one captured graph.
"""

from __future__ import annotations

import random

import numpy as np
import pytest
import torch

from tests.test_engine_gpu import SHAPES, VOCAB, Model, run_engine

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA GPU")
    return torch.device("cuda", 0)


def drafted_tree(rng, last, truth, size):
    """A tree of `size` nodes below `last`: some follow `truth`, the rest are wrong or continue wrong nodes."""
    tokens, parents, on_path = [last], [-1], [0]  # on_path[i]: how many true tokens node i's path holds
    while len(tokens) < size:
        up = rng.randrange(len(tokens))
        true_len = on_path[up]
        tok = truth[true_len] if true_len is not None and true_len < len(truth) and rng.random() < 0.7 else rng.randrange(VOCAB)
        ok = true_len is not None and true_len < len(truth) and tok == truth[true_len]
        tokens.append(tok)
        parents.append(up)
        on_path.append(true_len + 1 if ok else None)
    return tokens, parents


@pytest.mark.parametrize("shape", list(SHAPES))
@pytest.mark.parametrize("copy_on_write", [False, True])
def test_verified_trees_emit_the_greedy_stream(dev, shape, copy_on_write):
    from mini_inference_b200 import PagedKVCache
    from mini_inference_b200.sampler import GreedyLMHead

    rng = random.Random(21)
    model = Model(dev, seed=2, shape=SHAPES[shape])
    prompts = [[rng.randrange(VOCAB) for _ in range(rng.randint(1, 45))] for _ in range(5)]
    seqs, _, _ = run_engine(dev, model, [(p, 40) for p in prompts], num_blocks=60, max_seqs=5, budget=512, max_len=128)
    cache = PagedKVCache(2, model.hkv, model.d, num_blocks=60, block_size=16, max_seqs=5, max_len=128, dtype=model.dtype, device=dev,
                         enable_copy_on_write=copy_on_write)
    head = GreedyLMHead(model.lm, max_batch=256)
    slots = [cache.allocate(len(p) + 1) for p in prompts]
    ctx = cache.packed_prefill_context(slots, [len(p) for p in prompts])
    hidden = model.forward(torch.tensor([[t for p in prompts for t in p]], device=dev), ctx)
    ctx.commit()
    out = [[t] for t in head.tokens(hidden[0, ctx.last_index].contiguous())]
    accepted = 0
    for step in range(40):
        live = [i for i in range(5) if len(out[i]) < 30]
        if not live:
            break
        trees = [drafted_tree(rng, out[i][-1], seqs[i].output_token_ids[len(out[i]):len(out[i]) + 6],
                              rng.choice([1, 2, 7, 20, 70 if step == 1 else 12])) for i in live]
        ctx = cache.tree_context([slots[i] for i in live], [p for _, p in trees])
        ids = torch.tensor([t for toks, _ in trees for t in toks], device=dev)
        hidden = model.forward(ids[None], ctx)[0]
        new = ctx.accept(ids, head(hidden.contiguous()))
        for i, (toks, parents), row in zip(live, trees, new):
            want = seqs[i].output_token_ids[len(out[i]):len(out[i]) + len(row)]
            assert row[:len(want)] == want, (step, i)
            out[i] += row
            accepted += len(row) - 1
            assert cache.lengths[slots[i]] == len(prompts[i]) + len(out[i]) - 1
    cache.raise_device_errors()
    assert accepted > 50
    # A plain decode step goes on from what the trees left in the cache.
    ctx = cache.decode_context(slots)
    hidden = model.forward(torch.tensor([[o[-1]] for o in out], device=dev), ctx)
    ctx.commit()
    for i, tok in enumerate(head.tokens(hidden[:, -1].contiguous())):
        if len(out[i]) < 40:
            assert tok == seqs[i].output_token_ids[len(out[i])]


def test_tree_context_refusals(dev):
    from mini_inference_b200 import PagedKVCache

    cache = PagedKVCache(1, 2, 64, num_blocks=3, block_size=16, max_seqs=2, max_len=64, dtype=torch.float16, device=dev)
    slot = cache.allocate(20)
    cache.lengths[slot] = 20
    for slots, parents in (([slot], []), ([slot, slot], [[-1], [-1]]), ([slot], [[]]), ([slot], [[0]]), ([slot], [[-1, 1]]),
                           ([slot], [[-1, -1]]), ([slot], [[-1] * 1 + list(range(64))]), ([slot], [[-1] + [0] * 512])):
        with pytest.raises(ValueError):
            cache.tree_context(slots, parents)
    assert cache.tree_context([], []).accept(torch.zeros(0, dtype=torch.int64, device=dev), torch.zeros(0, dtype=torch.int64, device=dev)) == []
    with pytest.raises(ValueError, match="no room"):
        cache.tree_context([slot], [[-1] + list(range(40))])
    with pytest.raises(TypeError):
        x = torch.zeros(1, 14, 1, 64, device=dev)
        cache.tree_context([slot], [[-1]]).attend(0, x, x[:, :2], x[:, :2])


def dense_logits(model, cfg, tokens):
    """Float64 logits of every position of one sequence, from the model's weights."""
    from mini_inference_b200 import ops

    w = {k: v.double() for k, v in model.w.items()}
    r = cfg.rotary_dim or cfg.head_dim
    freq, factor = ops.rotary_frequencies(r, cfg.rope_theta, cfg.rope_scaling, model.device)
    n = len(tokens)
    angle = torch.arange(n, device=model.device, dtype=torch.float64)[:, None] * freq
    cos, sin = (angle.cos() * factor)[:, None], (angle.sin() * factor)[:, None]

    def rotate(x):
        x = x.clone()
        first, second = (slice(0, r, 2), slice(1, r, 2)) if cfg.rope_interleaved else (slice(0, r // 2), slice(r // 2, r))
        a, b = x[..., first].clone(), x[..., second].clone()
        x[..., first], x[..., second] = a * cos - b * sin, b * cos + a * sin
        return x

    def norm(x, name):
        return x / (x.pow(2).mean(-1, keepdim=True) + cfg.rms_norm_eps).sqrt() * w[name]

    x = w["embed_tokens.weight"][torch.tensor(tokens, device=model.device)]
    mask = torch.ones(n, n, dtype=torch.bool, device=model.device).tril()
    for i in range(cfg.num_layers):
        p = f"layers.{i}."
        qkv = norm(x, p + "input_norm.weight") @ w[p + "attn.qkv_proj.weight"].T + w[p + "attn.qkv_proj.bias"]
        heads = qkv.view(n, -1, cfg.head_dim)
        q, k, v = heads.split([cfg.num_heads, cfg.num_kv_heads, cfg.num_kv_heads], 1)
        q, k = rotate(q), rotate(k)
        k, v = (t.repeat_interleave(cfg.num_heads // cfg.num_kv_heads, 1) for t in (k, v))
        s = torch.einsum("qhd,khd->hqk", q, k) * cfg.head_dim ** -0.5
        o = torch.einsum("hqk,khd->qhd", s.masked_fill(~mask, -torch.inf).softmax(-1), v)
        x = x + o.reshape(n, -1) @ w[p + "attn.o_proj.weight"].T
        gate, up = (norm(x, p + "post_attn_norm.weight") @ w[p + "mlp.gate_up_proj.weight"].T).chunk(2, -1)
        x = x + (torch.nn.functional.silu(gate) * up) @ w[p + "mlp.down_proj.weight"].T
    return norm(x, "norm.weight") @ w["embed_tokens.weight"].T


@pytest.mark.parametrize("layout", ["plain", "yarn", "interleaved", "part", "part interleaved ntk"])
@pytest.mark.parametrize("speculative", [0, 5])
def test_engine_tokens_are_the_models_greedy_choices(dev, layout, speculative):
    """Every token within float16 rounding of the dense float64 forward's best logit (the engine tests' rule)."""
    from mini_inference_b200 import ops
    from mini_inference_b200.engine import EngineConfig, LLMEngine, SamplingParams
    from mini_inference_b200.model import Qwen2Config, Qwen2Model, init_random

    extra = {"plain": {}, "yarn": dict(rope_scaling=ops.RopeScaling("yarn", 4.0, 64)), "interleaved": dict(rope_interleaved=True),
             "part": dict(rotary_dim=32),
             "part interleaved ntk": dict(rotary_dim=48, rope_interleaved=True, rope_scaling=ops.RopeScaling("ntk", 2.0))}[layout]
    cfg = Qwen2Config(vocab_size=101, hidden_size=256, intermediate_size=320, num_layers=2, num_heads=6, num_kv_heads=2, head_dim=64,
                      max_position_embeddings=512, rope_theta=1e4, **extra)
    weights = init_random(cfg, seed=3, std=0.08, dtype=torch.float16, device=dev, unit_norms=True)
    model = Qwen2Model(cfg, weights)
    rng = random.Random(4)
    phrase = [rng.randrange(101) for _ in range(9)]
    prompts = [phrase * 3 + phrase[:4], [rng.randrange(101) for _ in range(50)], phrase[:5] * 2, [7]]
    engine = LLMEngine(model, EngineConfig(max_num_seqs=4, max_model_len=160, max_num_batched_tokens=256, kv_cache_tokens=640,
                                           speculative_tokens=speculative))
    seqs = engine.generate(prompts, SamplingParams(max_tokens=40, ignore_eos=True))
    steps = len(engine.step_stats)
    assert engine.runner.verify_tokens([], []) == []
    for s in seqs:
        assert len(s.output_token_ids) == 40
        rows = dense_logits(model, cfg, s.token_ids)[s.prompt_len - 1:-1]
        best = rows.amax(-1)
        got = rows.gather(1, torch.tensor(s.output_token_ids, device=dev)[:, None])[:, 0]
        assert (got >= best - 0.02 * best.abs().clamp(min=1.0)).all(), (best - got).max()
    assert steps == 40 if speculative == 0 else steps <= 40


def test_lookup_drafts():
    from mini_inference_b200.engine import EngineConfig, draft_by_lookup

    assert draft_by_lookup([1, 2, 3, 9, 1, 2, 3], 2) == [9, 1]
    assert draft_by_lookup([1, 2, 5, 2, 7, 2], 3) == [7, 2]  # the latest earlier occurrence
    assert draft_by_lookup([1, 2, 3], 4) == [] and draft_by_lookup([4], 4) == [] and draft_by_lookup([], 1) == []
    assert draft_by_lookup([1, 1, 1], 5) == [1]
    for bad in (-1, 64):
        with pytest.raises(ValueError):
            EngineConfig(speculative_tokens=bad)


@pytest.mark.parametrize("dtype,hq,hkv,d", [(torch.float16, 14, 2, 64), (torch.bfloat16, 28, 4, 128)])
def test_a_step_on_device_state_as_one_graph(dev, dtype, hq, hkv, d):
    """extend_tables, build_tree_metadata, then per layer rotary_append and tree_attention, and accept_tree,
    lengths and tables staying on the device: three steps eager, and as replays of one captured graph."""
    from mini_inference_b200 import ops

    layers, batch, bs, size, width = 2, 5, 16, 9, 4
    n = batch * size
    g = torch.Generator(device=dev).manual_seed(1)
    i32, i64 = dict(dtype=torch.int32, device=dev), dict(dtype=torch.int64, device=dev)
    parents = torch.tensor(([-1] + [(i - 1) // 2 for i in range(1, size)]) * batch, **i32)
    cu = torch.arange(0, n + 1, size, **i32)
    qkv = [torch.randn(n, (hq + 2 * hkv) * d, generator=g, device=dev).to(dtype) for _ in range(layers)]
    draft = torch.randint(0, 2, (n,), generator=g, **i64)
    target = torch.randint(0, 2, (n,), generator=g, **i64)
    freq, factor = ops.rotary_frequencies(d // 2, 1e4, ops.RopeScaling("linear", 2.0), dev)
    start = torch.tensor([0, 15, 16, 40, 31], **i32)

    class State:
        def __init__(self):
            g2 = torch.Generator(device=dev).manual_seed(2)
            self.k = torch.randn(layers, 41, hkv, bs, d, generator=g2, device=dev).to(dtype)
            self.v = torch.randn(layers, 41, hkv, bs, d, generator=g2, device=dev).to(dtype)
            self.pool = ops.make_pool(self.k, self.v)
            self.lengths, self.held = start.clone(), (start + bs - 1) // bs
            self.tables_t = torch.full((batch, 8), -1, **i32)
            at = 0
            for b in range(batch):
                h = int(self.held[b])
                self.tables_t[b, :h] = torch.arange(at, at + h, **i32)
                at += h
            self.tables = ops.make_tables(self.tables_t)
            self.free, self.head = torch.arange(at, 40, **i32), torch.zeros(1, **i32)
            self.new = torch.full((batch,), width, **i32)  # room for the longest path
            self.cu_seqlens, self.ctx_after = torch.empty(batch + 1, **i32), torch.empty(batch, **i32)
            self.mask, self.positions = torch.empty(n, 1, **i64), torch.empty(n, **i64)
            self.kn = torch.empty(layers, n, hkv, 1, d, dtype=dtype, device=dev)
            self.vn = torch.empty_like(self.kn)
            self.nodes, self.slots = ops.make_pool(self.kn, self.vn), torch.arange(n, **i64)
            self.ws = ops.tree_attention_workspace(self.pool, batch, dev)
            self.q = torch.empty(n, hq, d, dtype=dtype, device=dev)
            self.out = [torch.empty(n, hq, d, dtype=dtype, device=dev) for _ in range(layers)]
            self.counts, self.path = torch.empty(batch, **i32), torch.empty(batch, width, **i32)
            self.tokens, self.status = torch.empty(batch, width, **i64), torch.zeros(1, **i32)

        def step(self):
            ops.extend_tables(self.tables, self.lengths, self.new, self.held, self.free, self.head, bs, self.cu_seqlens,
                              self.ctx_after, status=self.status)
            ops.build_tree_metadata(parents, cu, self.lengths, self.mask, self.positions, self.status)
            for layer in range(layers):
                ops.rotary_append(self.nodes, layer, qkv[layer], self.positions, freq, hq, interleaved=True, attention_factor=factor,
                                  q_out=self.q, slot_mapping=self.slots, status=self.status)
                ops.tree_attention(self.pool, layer, self.tables, self.q, self.kn[layer, :, :, 0], self.vn[layer, :, :, 0], cu,
                                   self.lengths, self.mask, size, self.ws, out=self.out[layer], status=self.status)
            ops.accept_tree(self.pool, self.tables, parents, cu, draft, target, self.kn[:, :, :, 0], self.vn[:, :, :, 0],
                            self.lengths, self.counts, self.path, self.tokens, status=self.status)

        def values(self):
            torch.cuda.synchronize()
            ops.raise_device_errors(self.status)
            return [t.clone() for t in (self.k, self.v, self.lengths, self.held, self.head, self.tables_t, self.counts, self.path,
                                        self.tokens, self.positions, *self.out)]

    eager = State()
    want = []
    for _ in range(3):
        eager.step()
        want.append(eager.values())
    paths = want[0][6]
    assert (paths >= 1).all() and paths.max() > 1
    assert torch.equal(want[2][2], start + 3 * paths)  # the same tokens are accepted each time
    assert torch.equal(want[2][3], torch.maximum((start + 2 * paths + width + bs - 1) // bs, (start + bs - 1) // bs))

    warm, state = State(), State()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        warm.step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            state.step()
    torch.cuda.synchronize()
    for k in range(3):
        graph.replay()
        for a, b in zip(state.values(), want[k]):
            assert torch.equal(a, b)
