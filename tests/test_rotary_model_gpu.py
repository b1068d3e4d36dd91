"""Qwen2Model's rotary layouts: the keys it leaves in the cache, against float64 rotations of the projection's own rows."""

from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

from tests.test_rotary_gpu import check
from tests.test_speculative_engine_gpu import make_model, VOCAB

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA GPU")
    return torch.device("cuda", 0)


def layouts():
    from mini_inference_b200 import ops

    return {"yarn": dict(rope_scaling=ops.RopeScaling("yarn", 4.0, 64)), "linear": dict(rope_scaling=ops.RopeScaling("linear", 2.0)),
            "ntk": dict(rope_scaling=ops.RopeScaling("ntk", 8.0)), "interleaved": dict(rope_interleaved=True),
            "part": dict(rotary_dim=32), "part yarn": dict(rotary_dim=32, rope_scaling=ops.RopeScaling("yarn", 4.0, 64))}


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("layout", ["yarn", "linear", "ntk", "interleaved", "part", "part yarn"])
def test_cached_keys_are_rounded_once(dev, dtype, layout):
    """Prefill, a decode step and a verified tree: one rounding per element, whatever the frequencies."""
    from mini_inference_b200 import PagedKVCache, ops

    model = make_model(dev, dtype, **layouts()[layout])
    cfg = model.cfg
    cache = PagedKVCache(cfg.num_layers, cfg.num_kv_heads, cfg.head_dim, num_blocks=12, block_size=16, max_seqs=2, max_len=160, dtype=dtype,
                         device=dev)
    slot = cache.allocate(140)
    ids = torch.arange(130, device=dev) * 7 % VOCAB

    def keys(tokens, start):
        """The layer-0 keys of `tokens` from the cache, and what they are rotations of, as the model projects it."""
        n1, wqkv, bqkv = model.layers[0][:3]
        x = ops.add_rms_norm(F.embedding(tokens, model.embed), n1, cfg.rms_norm_eps).view(tokens.shape + (-1,))
        k = F.linear(x, wqkv, bqkv).view(tokens.numel(), -1, cfg.head_dim)[:, cfg.num_heads:cfg.num_heads + cfg.num_kv_heads]
        at = torch.arange(start, start + tokens.numel(), device=dev)
        blocks = torch.tensor(cache.block_tables[slot], device=dev)[at // 16]
        return cache.k[0, blocks, :, at % 16], k, at

    freq, factor = ops.rotary_frequencies(cfg.rotary_dim or 64, cfg.rope_theta, cfg.rope_scaling, dev)
    ctx = cache.packed_prefill_context([slot], [130])
    model(ids[None], ctx.positions[None], ctx)
    ctx.commit()
    got, k, at = keys(ids[None], 0)
    check(got, k, at, freq, cfg.rope_interleaved, factor)
    ctx = cache.decode_context([slot])
    last = torch.tensor([[5]], device=dev)
    model(last, ctx.positions[:, None], ctx)
    ctx.commit()
    got, k, at = keys(last, 130)
    check(got, k, at, freq, cfg.rope_interleaved, factor)
    ctx = cache.tree_context([slot], [[-1, 0, 1]])
    chain = torch.tensor([[9, 10, 11]], device=dev)
    model(chain, ctx.positions[None], ctx)
    assert ctx.accept(chain[0], chain[0] + 1) == [[10, 11, 12]]
    got, k, at = keys(chain, 131)
    check(got, k, at, freq, cfg.rope_interleaved, factor)
    cache.raise_device_errors()


def test_a_context_with_attend_alone_takes_scaled_tables(dev):
    """A context of someone else's, as the reference's: the model rotates by its tables."""
    model = make_model(dev, **layouts()["yarn"])
    seen = []

    class Attend:
        def attend(self, layer, q, k, v):
            seen.append((q.shape, k.shape))
            return torch.zeros_like(q)

    ids = torch.tensor([[1, 2, 3]], device=dev)
    out = model(ids, torch.arange(3, device=dev)[None], Attend())
    assert out.shape == (1, 3, 256) and seen == [((1, 6, 3, 64), (1, 2, 3, 64))] * 2
