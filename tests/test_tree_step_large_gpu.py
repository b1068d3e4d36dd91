"""Sizes at which extend_tables and rotary_append take another launch: many tokens, in place and apart.

extend_tables in place runs as one CTA up to 2,048 new tokens, as a cluster up to 16,384 and as two launches
beyond; rotary_append gives a thread four units from more than four tokens per SM on.
"""

from __future__ import annotations

import random

import pytest
import torch

from tests.test_rotary_gpu import check, setup
from tests.test_tree_step_gpu import check_extend

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA GPU")
    return torch.device("cuda", 0)


def batch_of(tokens, *, seed, bs=16, requests=64):
    """Arguments of check_extend: `requests` requests that bring `tokens` new tokens in all."""
    rng = random.Random(seed)
    cuts = sorted(rng.randint(0, tokens) for _ in range(requests - 1))
    new = [b - a for a, b in zip([0, *cuts], [*cuts, tokens])]
    lengths = [rng.randint(0, 300) for _ in new]
    held = [-(-a // bs) + rng.choice([0, 0, 1]) for a in lengths]
    cols = max(-(-(a + n) // bs) for a, n in zip(lengths, new)) + 2
    slots = rng.sample(range(requests + 3), requests)
    ids = rng.sample(range(100000), sum(held) + sum(new) // bs + 2 * requests)
    tables, at = [[-1] * cols for _ in range(requests + 3)], 0
    for s, h in zip(slots, held):
        tables[s][:h] = ids[at:at + h]
        at += h
    return dict(tables=tables, rows=slots, lengths=lengths, new=new, held=held, free=ids[at:], head=2, bs=bs, total=tokens)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("tokens", [2048, 2049, 16384, 16385, 40001])
def test_tables_of_many_tokens(dev, tokens, in_place):
    case = batch_of(tokens, seed=tokens)
    assert check_extend(dev, *case.values(), in_place=in_place)
    assert check_extend(dev, *{**case, "total": tokens + 77}.values(), in_place=in_place)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("tokens", [9000, 20000])
def test_refusals_of_many_tokens_change_nothing(dev, tokens, in_place):
    case = batch_of(tokens, seed=5)
    taken = sum(max(0, -(-(a + n) // 16) - h) for a, n, h in zip(case["lengths"], case["new"], case["held"]))
    few, narrow = case["free"][:2 + taken - 1], max(case["held"])
    wide = [n for n in case["new"]]
    wide[40] = -1
    for kw in (dict(free=few), dict(tables=[row[:narrow] for row in case["tables"]]), dict(total=tokens - 1), dict(new=wide),
               dict(head=len(case["free"]) + 1)):
        assert not check_extend(dev, *{**case, **kw}.values(), in_place=in_place), kw.keys()
    assert check_extend(dev, *{**case, "free": case["free"][:2 + taken]}.values(), in_place=in_place)


@pytest.mark.parametrize("dtype,hq,hkv,d,part", [(torch.bfloat16, 28, 4, 128, 128), (torch.float16, 14, 2, 64, 32),
                                                 (torch.float16, 3, 1, 80, 36)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("n", [592, 593, 2001])
def test_rotary_of_many_tokens(dev, dtype, hq, hkv, d, part, interleaved, n):
    from mini_inference_b200 import ops

    qkv, pos, k, v = setup(dev, dtype, hq, hkv, d, n, seed=n, blocks=130)
    freq, _ = ops.rotary_frequencies(part, 1e6, device=dev)
    slots = torch.randperm(130 * 16, device=dev)[:n]
    q, ko, vo = ops.rotary_append(ops.make_pool(k, v), 1, qkv, pos, freq, hq, interleaved=interleaved, k_out=True, v_out=True,
                                  slot_mapping=slots)
    heads = qkv.reshape(n, -1, d)
    check(q, heads[:, :hq], pos, freq, interleaved, 1.0)
    check(ko, heads[:, hq:hq + hkv], pos, freq, interleaved, 1.0)
    assert torch.equal(vo, heads[:, hq + hkv:])
    assert torch.equal(k[1, slots // 16, :, slots % 16], ko) and torch.equal(v[1, slots // 16, :, slots % 16], vo)
    assert (k[0] == 5).all() and (v[0] == 6).all()
