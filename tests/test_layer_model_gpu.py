"""Qwen2Model and the engine with head norms, position axes, media and experts, against the whole model in float64.

The operators have their own tests to the last rounding; here the question is whether the layer
calls them rightly (weights, order, positions, workspaces, contexts). A forward pass of L layers
rounds its activations about 16 times a layer by at most half a step of 2^-11 (float16): 16 L 2^-11
of the hidden states' size when errors add up and layers pass them on unchanged. Taken twice, for the
norms between, that is 1/32 for two layers; a layer called wrongly is off by the size of the values.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch
import torch.nn.functional as F

from mini_inference_b200 import PagedKVCache, ops
from mini_inference_b200.engine import EngineConfig, LLMEngine, Media, SamplingParams
from mini_inference_b200.model import Qwen2Config, Qwen2Model, init_random
from tests.test_media_positions_gpu import sequence
from tests.test_norm_rotary_gpu import check

pytestmark = pytest.mark.gpu
VOCAB = 211
LAYERS = 2
OFF = 1 / 32


def make_model(dtype=torch.float16, **kw):
    cfg = Qwen2Config(**(dict(vocab_size=VOCAB, hidden_size=192, intermediate_size=256, num_layers=LAYERS, num_heads=6, num_kv_heads=2,
                              head_dim=64, max_position_embeddings=1024, qk_norm=True, rope_sections=(8, 12, 12), num_experts=12,
                              experts_per_token=3, expert_intermediate_size=104, rope_theta=1e4) | kw))
    w = init_random(cfg, seed=3, std=0.08, dtype=dtype, device="cuda")
    for name, t in w.items():
        if name.endswith("norm.weight"):
            t.add_(1.0)
    return Qwen2Model(cfg, w)


def reference_hidden(model, tokens, positions, media=()):
    """Final hidden states [N, hidden] of one sequence, float64, every key attended to causally."""
    cfg, n = model.cfg, len(tokens)
    ids = torch.tensor(tokens, device="cuda")
    h = model.embed[ids].double()
    for a, rows in media:
        h[a:a + rows.shape[0]] = rows.double()
    freq, factor = ops.rotary_frequencies(cfg.rotary_dim or cfg.head_dim, cfg.rope_theta, cfg.rope_scaling)
    axes = ops.pair_axes(cfg.rope_sections, cfg.rope_sections_alternate).long() if cfg.rope_sections else None
    pos = torch.as_tensor(positions, device="cuda").double()  # [N, 3]
    angle = (pos[:, axes] if axes is not None else pos[:, :1]) * freq
    c, s = angle.cos()[:, None] * factor, angle.sin()[:, None] * factor

    def norm(x, w):
        return x / (x.square().mean(-1, keepdim=True) + cfg.rms_norm_eps).sqrt() * w.double()

    def turn(x):
        a, b = x.chunk(2, -1)
        return torch.cat([a * c - b * s, b * c + a * s], -1)

    causal = torch.ones(n, n, dtype=torch.bool, device="cuda").tril()
    for i, (n1, wqkv, bqkv, wo, n2, wgu, wd) in enumerate(model.layers):
        x = F.linear(norm(h, n1), wqkv.double(), bqkv.double()).view(n, -1, cfg.head_dim)
        q, k, v = x.split([cfg.num_heads, cfg.num_kv_heads, cfg.num_kv_heads], 1)
        if model.head_norms[i] is not None:
            q, k = norm(q, model.head_norms[i][0]), norm(k, model.head_norms[i][1])
        q, k = turn(q), turn(k)
        g = cfg.num_heads // cfg.num_kv_heads
        score = torch.einsum("qhd,khd->hqk", q, k.repeat_interleave(g, 1)) * cfg.head_dim ** -0.5
        score = score.masked_fill(~causal, -torch.inf).softmax(-1)
        h = h + F.linear(torch.einsum("hqk,khd->qhd", score, v.repeat_interleave(g, 1)).reshape(n, -1), wo.double())
        x = norm(h, n2)
        if model.routers:
            logits = x @ model.routers[i].double().T
            chosen = logits.topk(cfg.experts_per_token, -1).indices
            share = torch.zeros_like(logits).scatter(1, chosen, logits.softmax(-1).gather(1, chosen))
            if cfg.renormalize_experts:
                share = share / share.sum(-1, keepdim=True)
            gu = torch.einsum("nh,eih->nei", x, wgu.double())
            gate, up = gu.chunk(2, -1)
            h = h + torch.einsum("nei,ehi,ne->nh", F.silu(gate) * up, wd.double(), share)
        else:
            gate, up = F.linear(x, wgu.double()).chunk(2, -1)
            h = h + F.linear(F.silu(gate) * up, wd.double())
    return norm(h, model.norm)


def new_cache(model, max_media=4, **kw):
    cfg = model.cfg
    return PagedKVCache(cfg.num_layers, cfg.num_kv_heads, cfg.head_dim, num_blocks=80, block_size=16, max_seqs=4, max_len=256,
                        dtype=model.dtype, device="cuda", max_media=max_media, **kw)


def ids_of(n, seed):
    return np.random.default_rng(seed).integers(0, VOCAB, n).tolist()


def text(n):
    return np.repeat(np.arange(n)[:, None], 3, 1)


CONFIGS = {"all": {}, "norms": dict(rope_sections=None, num_experts=0), "axes": dict(qk_norm=False, num_experts=0),
           "experts": dict(qk_norm=False, rope_sections=None, renormalize_experts=False),
           "in turns, scaled": dict(rope_sections=(12, 10, 10), rope_sections_alternate=True,
                                    rope_scaling=ops.RopeScaling("yarn", 4.0, 64))}


@pytest.mark.parametrize("name", list(CONFIGS))
@torch.inference_mode()
def test_whole_model(name):
    """A packed prefill of two sequences, one with media, then decode steps and a verified tree."""
    model = make_model(**CONFIGS[name])
    several = model.cfg.rope_sections is not None
    cache = new_cache(model)
    spans = [(3, 1, 4, 5, 1), (30, 2, 3, 4, 2)] if several else []
    prompts = [ids_of(70, 1), ids_of(23, 2)]
    slots = [cache.allocate(len(p) + 8) for p in prompts]
    cache.set_media(slots[0], spans)
    ctx = cache.packed_prefill_context(slots, [70, 23])
    ids = torch.tensor([t for p in prompts for t in p], device="cuda")
    got = model(ids[None], ctx.positions[None], ctx)[0]
    ctx.commit()

    def compare(got, slot, tokens, last):
        pos = sequence(len(tokens), spans) if slot == 0 else text(len(tokens))
        want = reference_hidden(model, tokens, pos)[-last:]
        off = (got.double() - want).norm() / want.norm()
        assert off < OFF, off.item()

    compare(got[:70], 0, prompts[0], 70)
    compare(got[70:], 1, prompts[1], 23)
    for step in range(3):
        new = ids_of(2, 10 + step)
        ctx = cache.decode_context(slots)
        got = model(torch.tensor(new, device="cuda")[:, None], ctx.positions[:, None], ctx)
        ctx.commit()
        for i in range(2):
            prompts[i].append(new[i])
            compare(got[i], i, prompts[i], 1)
    # A chain of drafted tokens: its rows are those of the sequence that holds them.
    new = [ids_of(4, 50), ids_of(4, 51)]
    ctx = cache.tree_context(slots, [[-1, 0, 1, 2]] * 2)
    got = model(torch.tensor(new[0] + new[1], device="cuda")[None], ctx.positions[None], ctx)[0]
    for i in range(2):
        compare(got[4 * i:4 * i + 4], i, prompts[i] + new[i], 4)
    cache.raise_device_errors()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@torch.inference_mode()
def test_cached_keys_are_rounded_once(dtype):
    model = make_model(dtype)
    cfg, cache = model.cfg, new_cache(model)
    slot = cache.allocate(60)
    cache.set_media(slot, [(5, 1, 6, 7, 1)])
    ids = torch.tensor(ids_of(60, 4), device="cuda")
    ctx = cache.packed_prefill_context([slot], [60])
    model(ids[None], ctx.positions[None], ctx)
    n1, wqkv, bqkv = model.layers[0][:3]
    x = ops.add_rms_norm(F.embedding(ids[None], model.embed), n1, cfg.rms_norm_eps)
    k = F.linear(x, wqkv, bqkv).view(60, -1, 64)[:, 6:8]
    at = torch.arange(60, device="cuda")
    got = cache.k[0, torch.tensor(cache.block_tables[slot], device="cuda")[at // 16], :, at % 16]
    pos = torch.from_numpy(sequence(60, [(5, 1, 6, 7, 1)])).cuda().T
    check(got, k, pos, model.rotary.inv_freq, model.rotary.axes, model.head_norms[0][1], cfg.rms_norm_eps, False, 1.0)


@torch.inference_mode()
def test_a_slots_media_go_with_its_sequence():
    """Freed and taken again a slot has none; a fork has its parent's; refused spans change nothing."""
    model = make_model(num_experts=0)
    cache = new_cache(model, enable_copy_on_write=True)
    a = cache.allocate(40)
    cache.set_media(a, [(2, 1, 3, 3, 1)])
    cache.lengths[a] = 20
    b = cache.fork(a)
    for c in (cache.decode_context([a, b]), cache.packed_prefill_context([b, a], [2, 3])):
        assert c.axis_positions is not None and (c.axis_positions < c.positions).all()
    for bad in ([(2, 1, 3, 3)], [(2, 0, 3, 3, 1)], [(2, 1, 3, 3, -1)], [(5, 1, 2, 2, 1), (8, 1, 2, 2, 1)], [(0, 1, 1, 1, 1)] * 5,
                [(2**31, 1, 1, 1, 1)]):
        with pytest.raises(ValueError):
            cache.set_media(a, bad)
    assert cache.axis_positions([a], torch.tensor([20], device="cuda"), torch.tensor([a], dtype=torch.int32, device="cuda"),
                                None).tolist() == [[14]] * 3
    cache.free(a)
    assert cache.allocate(10) == a
    assert cache.decode_context([a]).axis_positions is None and cache.media_counts[a] == 0
    with pytest.raises(ValueError):
        new_cache(model, max_media=0).set_media(0, [(2, 1, 3, 3, 1)])


def check_streams(model, seqs):
    """Every output token is the float64 model's choice, or as good as it to what the roundings leave."""
    for s in seqs:
        tokens = s.prompt_token_ids + s.output_token_ids
        pos = sequence(len(tokens), [m.span for m in s.media])
        rows = [(m.start, m.rows.cuda().to(model.dtype)) for m in s.media if m.rows is not None]
        logits = reference_hidden(model, tokens, pos, rows) @ model.lm_head_weight.double().T
        logits = logits[len(s.prompt_token_ids) - 1:-1]
        mine = logits.gather(1, torch.tensor(s.output_token_ids, device="cuda")[:, None])[:, 0]
        # The hidden state is off by OFF of its size at most, and so a logit by that of |h| |w|.
        h, w = reference_hidden(model, tokens, pos, rows)[len(s.prompt_token_ids) - 1:-1], model.lm_head_weight.double()
        slack = 2 * OFF * h.norm(dim=-1) * w.norm(dim=-1).max()
        assert (mine >= logits.max(-1).values - slack).all()
        assert (mine == logits.max(-1).values).double().mean() > 0.7


def requests(model):
    g = torch.Generator().manual_seed(5)

    def rows(n):
        return torch.randn(n, model.cfg.hidden_size, generator=g).half()

    return [(ids_of(50, 21), [Media(4, 1, 5, 6, rows=rows(30))]), (ids_of(9, 22), []),
            (ids_of(80, 23), [Media(0, 2, 3, 4, 2, rows=rows(24)), Media(30, 1, 4, 4)]), (ids_of(17, 24), []),
            (ids_of(33, 25), [Media(10, 1, 2, 9, rows=rows(18))])]


@pytest.mark.parametrize("mode", ["eager", "graphs", "chunked", "speculative", "preempted"])
def test_engine(mode):
    model = make_model()
    kw = dict(max_num_seqs=4, max_model_len=160, max_num_batched_tokens=512, max_media=2, cuda_graphs=mode != "eager")
    if mode == "chunked":
        kw |= dict(chunked_prefill=True, max_num_batched_tokens=23)
    if mode == "speculative":
        kw |= dict(speculative_tokens=4)
    if mode == "preempted":
        kw |= dict(kv_cache_tokens=208)
    engine = LLMEngine(model, EngineConfig(**kw))
    ids = [engine.add_request(p, SamplingParams(max_tokens=24, ignore_eos=True), media=m) for p, m in requests(model)]
    while engine.has_unfinished_requests():
        engine.step()
    engine.check_device_errors()
    seqs = [engine.sequences[i] for i in ids]
    assert all(len(s.output_token_ids) == 24 for s in seqs)
    if mode == "preempted":
        assert any(s.num_preemptions for s in seqs)
    check_streams(model, seqs)


def test_engine_refusals():
    engine = LLMEngine(make_model(num_experts=0), EngineConfig(max_num_seqs=2, max_model_len=64, max_media=1, cuda_graphs=False))
    for media in ([Media(2, 1, 2, 2)] * 2, [Media(2, 1, 0, 2)], [Media(2, 1, 2, 2, -1)], [Media(6, 1, 2, 2)], [Media(-1, 1, 2, 2)],
                  [Media(2, 1, 2, 2, rows=torch.zeros(3, 192))]):
        with pytest.raises(ValueError):
            engine.add_request(list(range(10)), media=media)
    plain = LLMEngine(make_model(num_experts=0, rope_sections=None), EngineConfig(max_num_seqs=2, max_model_len=64, cuda_graphs=False))
    with pytest.raises(ValueError):
        plain.add_request(list(range(10)), media=[Media(2, 1, 2, 2)])
    with pytest.raises(ValueError):
        EngineConfig(max_media=1, enable_prefix_caching=True)


def test_an_experts_step_too_large_for_its_workspace_is_not_captured():
    model = make_model()
    model.expert_workspace(64)
    graph = torch.cuda.CUDAGraph()
    x = torch.zeros(1, device="cuda")
    with pytest.raises(RuntimeError, match="before capturing"):
        with torch.cuda.graph(graph):
            x.add_(1)
            model.expert_workspace(5000)


@torch.inference_mode()
def test_a_captured_step_keeps_its_workspace():
    """A larger step takes a larger workspace; the captured one's stays where its graph writes."""
    model = make_model()
    cache = new_cache(model)
    engine_like = [cache.allocate(40), cache.allocate(40)]
    ids = torch.tensor(ids_of(2, 3), device="cuda")
    from mini_inference_b200.cuda_graphs import GraphedDecoder
    graphs = GraphedDecoder(model, cache, 2)
    graphs.capture()
    first = model._expert_workspaces[-1]
    model.expert_workspace(5000)
    assert model._expert_workspaces[-1] is not first and model._expert_workspaces[0] is first
    model._expert_workspaces[-1].fill_(0)
    for s in engine_like:
        cache.lengths[s] = 0
    logits = graphs.decode(engine_like, ids.tolist())
    for s in engine_like:
        cache.lengths[s] = 0
    ctx = cache.decode_context(engine_like)
    want = model.compute_logits(model(ids[:, None], ctx.positions[:, None], ctx)[:, -1]).float()
    assert torch.equal(logits, want)
    assert not first[:6200].any()
