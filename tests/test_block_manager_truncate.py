"""pkv_bm_truncate: blocks behind a sequence's tokens go back to the free pool, as they came. No GPU needed."""

from __future__ import annotations

import random

import pytest

from mini_inference_b200.cache import NativeBlockManager


def test_growing_and_truncating_leaves_the_pool_as_it_was():
    bm = NativeBlockManager(20, 16, 4, 200, False)
    a, b = bm.allocate(20), bm.allocate(33)
    before = bm.state()
    for tokens in (21, 32, 33, 64, 200):
        assert bm.ensure_capacity(a, tokens)
        bm.truncate(a, 20)
        assert bm.state() == before
    assert bm.ensure_capacity(a, 100) and bm.num_blocks_held(a) == 7 and bm.num_blocks_held(b) == 3
    bm.truncate(a, 100)
    assert bm.num_blocks_held(a) == 7
    bm.truncate(a, 96)
    assert bm.num_blocks_held(a) == 6 and bm.num_free_blocks == 20 - 9
    bm.truncate(a, 0)  # its length is zero: nothing was committed
    assert bm.num_blocks_held(a) == 0
    bm.free(a)
    bm.free(b)
    assert bm.num_free_blocks == 20


def test_shared_blocks_stay_with_the_other_sequence():
    bm = NativeBlockManager(8, 16, 3, 100, False)
    a = bm.allocate(40)
    bm.set_length(a, 10)
    c = bm.fork(a)
    bm.truncate(c, 10)
    assert bm.table(c) == bm.table(a)[:1] and bm.num_blocks_held(a) == 3 and bm.num_free_blocks == 5
    bm.free(a)
    assert bm.num_free_blocks == 7


def test_refusals():
    bm = NativeBlockManager(8, 16, 2, 100, False)
    slot = bm.allocate(40)
    bm.set_length(slot, 17)
    with pytest.raises(ValueError):
        bm.truncate(slot, 16)
    for bad in (slot + 1, -1, 7):
        with pytest.raises(KeyError):
            bm.truncate(bad, 40)
        with pytest.raises(KeyError):
            bm.num_blocks_held(bad)
    assert bm.num_blocks_held(slot) == 3


def test_every_block_has_one_owner():
    rng = random.Random(3)
    bm = NativeBlockManager(30, 4, 6, 60, True)
    live = {}
    for _ in range(2000):
        what = rng.random()
        if what < 0.3 and len(live) < 6:
            ids = [rng.randrange(3) for _ in range(rng.randint(1, 20))]
            if bm.can_allocate(len(ids)):
                slot = bm.allocate(len(ids), ids)
                bm.set_length(slot, len(ids))
                bm.register_prefix(slot, ids)
                live[slot] = len(ids)
        elif what < 0.6 and live:
            bm.ensure_capacity(rng.choice(list(live)), rng.randint(1, 60))
        elif what < 0.85 and live:
            slot = rng.choice(list(live))
            bm.truncate(slot, live[slot] + rng.randint(0, 9))
        elif live:
            slot = rng.choice(list(live))
            bm.free(slot)
            del live[slot]
        refs, free = bm.ref_counts(), bm.free_block_order()
        held = [b for s in live for b in bm.table(s)]
        assert [held.count(b) for b in range(30)] == refs
        assert sorted(free) == [b for b in range(30) if refs[b] == 0]
        assert all(bm.num_blocks_held(s) * 4 >= n for s, n in live.items())
