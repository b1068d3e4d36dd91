"""ops.media_positions (positions on three axes of prompts with images and video) against a plain loop."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from mini_inference_b200 import ops

pytestmark = pytest.mark.gpu


def sequence(length, spans):
    """Every token's three positions, written out one after another."""
    out, at, i = [], 0, 0
    spans = {s[0]: s for s in spans}
    while i < length:
        if i in spans:
            _, frames, h, w, step = spans[i]
            out += [(at + f * step, at + y, at + x) for f in range(frames) for y in range(h) for x in range(w)]
            i += frames * h * w
            at += max((frames - 1) * step + 1, h, w)
        else:
            out.append((at,) * 3)
            i, at = i + 1, at + 1
    return np.array(out[:length], np.int64).reshape(-1, 3)


def table(rows, cap=None):
    cap = cap or max(1, max(map(len, rows)))
    t = np.zeros((len(rows), cap, 5), np.int32)
    for r, spans in enumerate(rows):
        if spans:
            t[r, :len(spans)] = spans
    return torch.from_numpy(t).cuda(), torch.tensor([len(r) for r in rows], dtype=torch.int32, device="cuda")


def draw(rng, spans):
    rows, at = [], 0
    for _ in range(spans):
        at += int(rng.integers(0, 9))
        frames, h, w = int(rng.choice([1, 1, 3])), int(rng.integers(1, 9)), int(rng.integers(1, 9))
        rows.append((at, frames, h, w, int(rng.integers(0, 5))))
        at += frames * h * w
    return rows, at


def test_the_loop_itself():
    # Text of 2, an image of 2 x 3, text of 1: the text goes on at 2 + 3.
    assert sequence(9, [(2, 1, 2, 3, 1)]).tolist() == [[0] * 3, [1] * 3, [2, 2, 2], [2, 2, 3], [2, 2, 4], [2, 3, 2], [2, 3, 3],
                                                      [2, 3, 4], [5] * 3]


@pytest.mark.parametrize("batch,spans", [(1, 0), (1, 1), (5, 3), (40, 12)])
def test_packed(batch, spans):
    rng = np.random.default_rng(batch)
    rows, want, pos, counts = [], [], [], []
    for b in range(batch):
        r, end = draw(rng, int(rng.integers(0, spans + 1)))
        length = end + int(rng.integers(0, 30))
        first = int(rng.integers(0, length + 1)) if b % 3 else 0  # a chunk from the middle on, perhaps empty
        n = int(rng.integers(0, length - first + 1))
        rows.append(r)
        want.append(sequence(length, r)[first:first + n])
        pos.append(np.arange(first, first + n))
        counts.append(n)
    order = rng.permutation(batch)  # sequences' rows in the table
    placed = [None] * batch
    for b in range(batch):
        placed[order[b]] = rows[b]
    media, counts_dev = table(placed, cap=spans + 2)
    cu = torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device="cuda")
    total = int(cu[-1])
    pos = torch.from_numpy(np.concatenate(pos + [np.arange(7)])).cuda()  # 7 tokens behind the last sequence
    out = torch.full((3, total + 7), -5, dtype=torch.int64, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = ops.media_positions(pos, media, counts_dev, torch.tensor(order, dtype=torch.int32, device="cuda"), cu, out=out,
                              status=status)
    ops.raise_device_errors(status)
    assert got is out or torch.equal(got, out)
    assert np.array_equal(out[:, :total].T.cpu().numpy(), np.concatenate(want))
    assert (out[:, total:] == -5).all()


@pytest.mark.parametrize("batch", [1023, 1024, 1025, 2100])
def test_many_sequences(batch):
    """Chunks of 0 to 2 tokens; rows of 0 to 9 spans, which the kernel reads four at a time."""
    rng = np.random.default_rng(batch)
    rows, want, pos, counts = [], [], [], []
    for b in range(batch):
        r, end = draw(rng, b % 10)
        n = int(rng.integers(0, 3))
        first = int(rng.integers(0, end + 3))
        rows.append(r)
        want.append(sequence(first + n, r)[first:])
        pos.append(np.arange(first, first + n))
        counts.append(n)
    media, counts_dev = table(rows, cap=9 + batch % 2)
    cu = torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = ops.media_positions(torch.from_numpy(np.concatenate(pos)).cuda(), media, counts_dev, None, cu, status=status)
    ops.raise_device_errors(status)
    assert np.array_equal(got.T.cpu().numpy(), np.concatenate(want))


@pytest.mark.parametrize("wrong,at,reported", [(4, 100, True), (7, 100, True), (4, 6, False), (8, 100, True)])
def test_a_later_span_is_wrong(wrong, at, reported):
    """Reported by the tokens behind it: one in the second span does not read so far."""
    spans = [(4 * i, 1, 1, 3, 1) for i in range(9)]
    spans[wrong] = (4 * wrong, 1, 0, 3, 1)
    media, counts = table([spans])
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    ops.media_positions(torch.tensor([at], device="cuda"), media, counts, status=status)
    assert bool(status.item()) == reported


def test_one_token_each():
    """A decode batch: no cu_seqlens; padding rows (-1) have no media; rows given or not."""
    media, counts = table([[(2, 1, 4, 5, 1)], [], [(0, 2, 3, 3, 4), (18, 1, 1, 1, 1)]])
    pos = torch.tensor([30, 7, 19, 5], device="cuda")
    rows = torch.tensor([0, 1, 2, -1], dtype=torch.int32, device="cuda")
    got = ops.media_positions(pos, media, counts, rows)
    want = [sequence(31, [(2, 1, 4, 5, 1)])[30], (7, 7, 7), sequence(20, [(0, 2, 3, 3, 4), (18, 1, 1, 1, 1)])[19], (5, 5, 5)]
    assert got.T.tolist() == [list(map(int, w)) for w in want]
    assert torch.equal(ops.media_positions(pos[:3], media, counts), got[:, :3])
    wide = torch.zeros(3, 10, dtype=torch.int64, device="cuda")
    ops.media_positions(pos, media, counts, rows, out=wide[:, 2:6])
    assert torch.equal(wide[:, 2:6], got) and not wide[:, :2].any() and not wide[:, 6:].any()
    assert ops.media_positions(pos[:0], media, counts, rows[:0]).shape == (3, 0)
    none = torch.zeros(0, 0, 5, dtype=torch.int32, device="cuda")
    assert torch.equal(ops.media_positions(pos, none, counts[:0], rows.clamp(max=-1)), pos.expand(3, -1))


def test_large_numbers():
    """Indexes and sizes past 32 bits in sum."""
    media, counts = table([[(2**31 - 1, 2**20, 2**10, 2**10, 7)]])
    far = 2**31 - 1 + 5 * 2**20 + 3 * 2**10 + 9
    pos = torch.tensor([far, 2**62], device="cuda")
    got = ops.media_positions(pos, media, counts, torch.zeros(2, dtype=torch.int32, device="cuda"))
    a = 2**31 - 1
    size, ahead = 2**40, (2**20 - 1) * 7 + 1
    assert got.T.tolist() == [[a + 35, a + 3, a + 9], [2**62 - size + ahead] * 3]


@pytest.mark.parametrize("bad", [dict(spans=[(5, 1, 2, 2, 1), (8, 1, 2, 2, 1)]), dict(spans=[(0, 0, 2, 2, 1)]),
                                 dict(spans=[(0, 1, -2, 2, 1)]), dict(spans=[(0, 2, 2, 2, -1)]), dict(spans=[(-1, 1, 2, 2, 1)]),
                                 dict(count=2), dict(count=-1), dict(row=1)])
def test_reports(bad):
    media, counts = table([bad.get("spans", [(3, 1, 2, 2, 1)])])
    if "count" in bad:
        counts[0] = bad["count"]
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    ops.media_positions(torch.tensor([20], device="cuda"), media, counts,
                        torch.tensor([bad.get("row", 0)], dtype=torch.int32, device="cuda"), status=status)
    with pytest.raises(IndexError):
        ops.raise_device_errors(status)


def test_refusals():
    media, counts = table([[(3, 1, 2, 2, 1)]])
    pos, rows = torch.tensor([20], device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    ok = dict(positions=pos, media=media, media_counts=counts, seq_rows=rows)
    for kw in (dict(positions=pos.int()), dict(media=media[:, :, :4].contiguous()), dict(media=media.long()),
               dict(media_counts=counts[:0]), dict(seq_rows=rows[:0]), dict(cu_seqlens=rows[:0]),
               dict(out=torch.empty(2, 1, dtype=torch.int64, device="cuda")), dict(seq_rows=None, media=media[:0]),
               dict(out=torch.empty(3, 1, device="cuda")), dict(seq_rows=rows.cpu())):
        with pytest.raises(ValueError):
            ops.media_positions(**{**ok, **kw})
