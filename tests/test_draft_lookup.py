"""Drafts by lookup (pkv_draft_by_lookup, pkv_sched_draft) against a plain restatement. No GPU needed."""

from __future__ import annotations

import ctypes
import random
import time
from types import SimpleNamespace

import numpy as np
import pytest

from mini_inference_b200 import PkvError, _lib
from mini_inference_b200.engine import draft_by_lookup, SamplingParams, Sequence
from mini_inference_b200.scheduler import Scheduler, SequenceStatus

L = _lib.lib


def plain(ids, count, longest=3):
    """The longest tail first, its occurrences from the end backwards."""
    n = len(ids)
    for size in range(min(longest, n - 1), 0, -1):
        for at in range(n - size - 1, -1, -1):
            if ids[at:at + size] == ids[n - size:]:
                return ids[at + size:at + size + count]
    return []


def test_against_the_plain_form():
    rng = random.Random(1)
    for _ in range(3000):
        ids = [rng.randrange(rng.choice([1, 2, 3, 8, 40])) - 1 for _ in range(rng.randint(0, 40))]
        count, longest = rng.randint(0, 9), rng.randint(0, 5)
        assert draft_by_lookup(ids, count, longest) == plain(ids, count, longest), (ids, count, longest)
    assert draft_by_lookup([5, 1 << 40, 7, 1 << 40], 2) == [7, 1 << 40]
    assert draft_by_lookup([1, 1], -3) == [] and draft_by_lookup([1, 2, 1], 1 << 60) == [2, 1]


def make_scheduler(texts, max_tokens=50):
    from mini_inference_b200 import PagedKVCache
    import torch

    longest = max(map(len, texts)) + 60
    cache = PagedKVCache(1, 1, 64, num_blocks=len(texts) * (longest // 16 + 2), block_size=16, max_seqs=len(texts), max_len=longest,
                         dtype=torch.float16, device="cpu")
    sched = Scheduler(SimpleNamespace(max_num_seqs=len(texts), max_num_batched_tokens=1 << 24, max_model_len=longest,
                                      scheduling="continuous"), cache)
    seqs = [Sequence(i, list(t), SamplingParams(max_tokens=max_tokens, ignore_eos=True), 0.0) for i, t in enumerate(texts)]
    for s in seqs:
        sched.add(s)
    assert sched.schedule().prefills == seqs
    return sched, seqs


def test_the_schedulers_own_tokens():
    rng = random.Random(2)
    sched, seqs = make_scheduler([[rng.randrange(4) for _ in range(rng.randint(1, 30))] for _ in range(12)])
    for step in range(20):
        sched.append_tokens(seqs, [rng.randrange(4) for _ in seqs], 0.0)
        counts = [rng.randint(-1, 6) for _ in seqs]
        assert sched.draft(seqs, counts) == [plain(s.token_ids, c) if c > 0 else [] for s, c in zip(seqs, counts)]
    assert sched.draft([], []) == [] and sched.draft(seqs[:2], [0, -4]) == [[], []]
    sched.abort(seqs[0], 0.0)
    assert seqs[0].status is SequenceStatus.FINISHED
    with pytest.raises(PkvError):
        sched.draft(seqs, [1] * 12)


def test_long_texts_cost_little():
    """64 sequences of 32K tokens whose last token has not occurred before: a step's drafts in well under 100 ms."""
    sched, seqs = make_scheduler([range(32768)] * 64)
    t0 = time.process_time()
    assert sched.draft(seqs, [8] * 64) == [[]] * 64
    assert time.process_time() - t0 < 0.1


def test_refusals():
    text = np.array([1, 2, 1], np.int64)
    out, got = np.zeros(4, np.int64), ctypes.c_int32()

    def call(tokens=text.ctypes.data, n=3, longest=3, count=4, dst=out.ctypes.data, n_out=ctypes.byref(got)):
        return L.pkv_draft_by_lookup(tokens, n, longest, count, dst, n_out)

    assert call() == _lib.PKV_OK and got.value == 2 and out[:2].tolist() == [2, 1]
    for kw in (dict(tokens=None), dict(n=-1), dict(longest=-1), dict(count=-1), dict(dst=None), dict(n_out=None)):
        assert call(**kw) == _lib.PKV_ERR_INVALID_ARGUMENT, kw
    assert call(tokens=None, n=0) == _lib.PKV_OK and got.value == 0
    assert call(dst=None, count=0) == _lib.PKV_OK and got.value == 0
    sched, seqs = make_scheduler([[1, 2, 1]])
    ids, counts, n_out = np.array([0], np.int64), np.array([2], np.int32), np.zeros(1, np.int32)

    def batch(h=sched._h, i=ids.ctypes.data, c=counts.ctypes.data, n=1, longest=3, dst=out.ctypes.data, stride=2, g=n_out.ctypes.data):
        return L.pkv_sched_draft(h, i, c, n, longest, dst, stride, g)

    assert batch() == _lib.PKV_OK and n_out[0] == 2 and out[:2].tolist() == [2, 1]
    for kw in (dict(h=None), dict(i=None), dict(c=None), dict(n=-1), dict(longest=-1), dict(dst=None), dict(stride=-1), dict(g=None),
               dict(stride=1)):
        assert batch(**kw) == _lib.PKV_ERR_INVALID_ARGUMENT, kw
    assert batch(n=0, i=None) == _lib.PKV_OK
