"""The steps around tree attention on the GPU: tables from lengths, tree metadata, acceptance. All exact.

Each kernel against a plain restatement in Python integers (``extend``, ``metadata``, ``accept`` below).
"""

from __future__ import annotations

import random

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA GPU")
    return torch.device("cuda", 0)


def i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


# ---------------------------------------------------------------- tables from lengths

def extend(tables, rows, lengths, new, held, free, head, bs, total):
    """(tables, cu, ctx, positions, slots, held, head, ok)"""
    tables = [list(r) for r in tables]
    need = [0 if r < 0 else max(h, -(-(a + n) // bs)) for r, a, n, h in zip(rows, lengths, new, held)]
    cu = [0]
    for n in new:
        cu.append(cu[-1] + max(n, 0))
    ok = all(n >= 0 for n in new) and cu[-1] <= total and all(
        r < 0 or (r < len(tables) and a >= 0 and 0 <= h <= len(tables[0]) and m <= len(tables[0]))
        for r, a, h, m in zip(rows, lengths, held, need))
    fresh = [max(0, m - h) if r >= 0 else 0 for r, m, h in zip(rows, need, held)]
    ok = ok and head >= 0 and sum(fresh) <= max(0, len(free) - head)
    cu = [min(c, total) for c in cu]
    if not ok:
        ctx = [max(a, 0) if r >= 0 else 0 for r, a in zip(rows, lengths)]
        return tables, cu, ctx, [0] * total, [-1] * total, list(held), head, False
    positions, slots, at = [0] * total, [-1] * total, head
    for b, r in enumerate(rows):
        for i in range(fresh[b]):
            tables[r][held[b] + i] = free[at]
            at += 1
        for i in range(new[b]):
            if r >= 0:
                p = lengths[b] + i
                positions[cu[b] + i] = p
                slots[cu[b] + i] = tables[r][p // bs] * bs + p % bs
    ctx = [a + n if r >= 0 else 0 for r, a, n in zip(rows, lengths, new)]
    return tables, cu, ctx, positions, slots, [h + f for h, f in zip(held, fresh)], at, True


def run_extend(dev, tables, rows, lengths, new, held, free, head, bs, total, in_place):
    from mini_inference_b200 import ops

    b = len(lengths)
    t = i32(tables, dev)
    args = [i32(x, dev) for x in (lengths, new, held, free)]
    hd = i32([head], dev)
    cu, ctx = i32([7] * (b + 1), dev), args[0] if in_place else i32([7] * b, dev)
    pos, slots = (torch.full((total,), 7, dtype=torch.int64, device=dev) for _ in range(2))
    held_out, head_out = (None, None) if in_place else (i32([7] * b, dev), i32([7], dev))
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    ops.extend_tables(ops.make_tables(t, i32(rows, dev)), args[0], args[1], args[2], args[3], hd, bs, cu, ctx, pos, slots,
                      held_out=held_out, free_head_out=head_out, status=status)
    got = (t.tolist(), cu.tolist(), ctx.tolist(), pos.tolist(), slots.tolist(),
           (args[2] if in_place else held_out).tolist(), (hd if in_place else head_out).item())
    return got, status


def check_extend(dev, *case, in_place=False):
    from mini_inference_b200 import ops

    want = extend(*case)
    got, status = run_extend(dev, *case, in_place)
    assert got == tuple(want[:7])
    if want[7]:
        ops.raise_device_errors(status)
    else:
        assert status.item() in (2, 5)
    return want[7]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("batch,most_new,most_len,bs", [(1, 1, 0, 16), (1, 40, 100, 16), (5, 3, 33, 16), (33, 1, 2000, 16),
                                                        (300, 70, 500, 16), (64, 9, 50, 1), (31, 40, 90, 7),
                                                        (1500, 2, 60, 16), (4096, 3, 40, 16)])
def test_tables_from_lengths(dev, batch, most_new, most_len, bs, in_place):
    rng = random.Random(batch + bs)
    lengths = [rng.randint(0, most_len) for _ in range(batch)]
    new = [rng.randint(0, most_new) for _ in range(batch)]
    spare = [rng.choice([0, 0, 1]) for _ in range(batch)]  # some already hold a block more
    held = [-(-a // bs) + s for a, s in zip(lengths, spare)]
    cols = -(-(most_len + most_new) // bs) + 2
    slots = rng.sample(range(batch + 7), batch)
    rows = [-1 if batch > 4 and rng.random() < 0.1 else s for s in slots]
    ids = rng.sample(range(100000), sum(held) + batch * cols)
    tables, at = [[-1] * cols for _ in range(batch + 7)], 0
    for s, h in zip(slots, held):
        tables[s][:h] = ids[at:at + h]
        at += h
    free = ids[at:] + [1]
    total = sum(new) + rng.choice([0, 5])
    assert check_extend(dev, tables, rows, lengths, new, held, free, min(3, len(free) - 1), bs, max(total, 1),
                        in_place=in_place)


def test_tables_all_or_nothing(dev):
    tables = [[3, -1, -1], [4, 5, -1]]
    ok = dict(tables=tables, rows=[0, 1], lengths=[10, 20], new=[10, 4], held=[1, 2], free=[9, 8, 7], head=0, bs=16, total=14)

    def case(**kw):
        return check_extend(dev, *{**ok, **kw}.values())

    assert case()
    assert case(free=[9], head=0)
    for kw in (dict(free=[9], head=1), dict(head=3), dict(head=5), dict(new=[10, 30]), dict(new=[10, -1]), dict(new=[39, 4]),
               dict(lengths=[-1, 20]), dict(held=[4, 2]), dict(held=[-1, 2]), dict(rows=[0, 2]), dict(total=13), dict(head=-1),
               dict(lengths=[10, 2**31 - 2])):
        assert not case(**kw), kw


def test_tables_of_no_request_and_without_slots(dev):
    from mini_inference_b200 import ops

    empty = i32([], dev)
    cu, head = i32([7], dev), i32([1], dev)
    slots = torch.full((3,), 7, dtype=torch.int64, device=dev)
    ops.extend_tables(ops.make_tables(i32([[1]], dev)), empty, empty, empty, i32([4, 5], dev), head, 16, cu, empty, slots.clone(), slots)
    assert cu.tolist() == [0] and head.item() == 1 and slots.tolist() == [-1] * 3
    t, held, ctx = i32([[-1, -1]], dev), i32([0], dev), i32([0], dev)
    ops.extend_tables(ops.make_tables(t), i32([0], dev), i32([20], dev), held, i32([4, 5, 6], dev), head, 16, i32([0, 0], dev), ctx)
    assert t.tolist() == [[5, 6]] and held.item() == 2 and head.item() == 3 and ctx.item() == 20


# ---------------------------------------------------------------- tree metadata

def metadata(parents):
    masks, depths = [], []
    for i, up in enumerate(parents):
        masks.append((masks[up] if up >= 0 else 0) | 1 << i)
        depths.append(depths[up] + 1 if up >= 0 else 0)
    return masks, depths


def random_tree(rng, n, kind):
    if kind == "chain":
        return [i - 1 for i in range(n)]
    if kind == "star":
        return [-1] + [0] * (n - 1) if n else []
    if kind == "forest":
        return [rng.randint(-1, i - 1) if rng.random() < 0.8 else -1 for i in range(n)]
    return [-1] + [rng.randint(max(0, i - 6), i - 1) for i in range(1, n)] if n else []


@pytest.mark.parametrize("kind", ["random", "chain", "star", "forest"])
@pytest.mark.parametrize("sizes,words,behind", [([1], 1, 0), ([8], 1, 0), ([64, 1, 0, 63], 1, 3), ([65, 128, 2], 2, 0),
                                                ([512, 300, 511], 8, 1), ([40] * 256, 1, 0), ([5], 8, 2)])
def test_tree_metadata(dev, kind, sizes, words, behind):
    from mini_inference_b200 import ops

    rng = random.Random(sum(sizes))
    trees = [random_tree(rng, n, kind) for n in sizes]
    ctx = [rng.randint(0, 10**6) for _ in sizes]
    n = sum(sizes) + behind
    cu = [0]
    for s in sizes:
        cu.append(cu[-1] + s)
    parents = i32([p for t in trees for p in t] + [0] * behind, dev)
    mask = torch.full((n, words), 7, dtype=torch.int64, device=dev)
    positions = torch.full((n,), 7, dtype=torch.int64, device=dev)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    ops.build_tree_metadata(parents, i32(cu, dev), i32(ctx, dev), mask, positions, status)
    ops.raise_device_errors(status)
    want_m, want_p = [], []
    for t, c in zip(trees, ctx):
        masks, depths = metadata(t)
        want_m += masks
        want_p += [c + d for d in depths]
    got = [sum((w & (2**64 - 1)) << 64 * i for i, w in enumerate(r)) for r in mask.tolist()]
    assert got == want_m + [0] * behind
    assert positions.tolist() == want_p + [0] * behind


def test_bad_trees_are_reported(dev):
    from mini_inference_b200 import ops

    def run(parents, cu, words=1):
        n = len(parents)
        mask, pos = torch.zeros(n, words, dtype=torch.int64, device=dev), torch.zeros(n, dtype=torch.int64, device=dev)
        status = torch.zeros(1, dtype=torch.int32, device=dev)
        ops.build_tree_metadata(i32(parents, dev), i32(cu, dev), i32([0] * (len(cu) - 1), dev), mask, pos, status)
        with pytest.raises(IndexError):
            ops.raise_device_errors(status)
        return mask, pos

    mask, pos = run([-1, 0, 2], [0, 3])  # its own parent: taken as a root
    assert mask.flatten().tolist() == [1, 3, 4] and pos.tolist() == [0, 1, 0]
    run([-1, 5, 1], [0, 3])
    run([-1, -2, 1], [0, 3])
    run([-1, 0, 1], [0, 4])
    run([-1, 0, 1], [2, 0])
    mask, pos = run([-1] + list(range(69)), [0, 70])  # 70 nodes, one word
    assert mask[64:].eq(0).all() and pos[:64].tolist() == list(range(64))


# ---------------------------------------------------------------- acceptance

def accept(parents, draft, target, width):
    path = [0] if parents else []
    while path and len(path) < width:
        hits = [j for j in range(path[-1] + 1, len(parents)) if parents[j] == path[-1] and draft[j] == target[path[-1]]]
        if not hits:
            break
        path.append(hits[0])
    return path


@pytest.mark.parametrize("dtype,hkv,d,layers", [(torch.float16, 2, 64, 24), (torch.bfloat16, 4, 128, 3), (torch.float16, 1, 36, 2),
                                                (torch.bfloat16, 3, 64, 1)])
@pytest.mark.parametrize("sizes,width,in_place", [([1], 4, False), ([8, 0, 20, 64], 8, True), ([30] * 130, 5, False),
                                                  ([512, 3], 64, True)])
def test_acceptance(dev, dtype, hkv, d, layers, sizes, width, in_place):
    from mini_inference_b200 import ops

    rng = random.Random(sum(sizes) + d)
    bs, batch, n = 16, len(sizes), sum(sizes)
    trees = [random_tree(rng, s, "chain" if s == 512 else "random") for s in sizes]
    drafts = [[rng.randint(0, 2) for _ in range(s)] for s in sizes]  # few tokens: equal siblings, long paths
    targets = [[rng.randint(0, 2) if s != 512 else t[min(i + 1, s - 1)] for i in range(s)] for s, t in zip(sizes, drafts)]
    ctx = [rng.randint(0, 50) for _ in sizes]
    cols = (50 + 64) // bs + 2
    order = torch.randperm(batch * cols)
    slots = rng.sample(range(batch + 3), batch)
    table = torch.full((batch + 3, cols), -1, dtype=torch.int32)
    for b, s in enumerate(slots):
        table[s] = order[b * cols:(b + 1) * cols].int()
    rows = [-1 if batch > 3 and b == 2 else s for b, s in enumerate(slots)]
    k = torch.randn(layers, batch * cols + 1, hkv, bs, d, device=dev).to(dtype)
    v = torch.randn_like(k)
    kn = torch.randn(layers, n, hkv, d, device=dev).to(dtype)
    wide = torch.randn(layers, n, 3 * hkv * d, device=dev).to(dtype)
    vn = wide[:, :, hkv * d:2 * hkv * d].view(layers, n, hkv, d)  # columns of wider rows
    want_k, want_v = k.clone(), v.clone()
    cu = [0]
    for s in sizes:
        cu.append(cu[-1] + s)
    lens = i32(ctx, dev)
    counts, path = i32([7] * batch, dev), torch.full((batch, width), 7, dtype=torch.int32, device=dev)
    tokens = torch.full((batch, width), 7, dtype=torch.int64, device=dev)
    out = None if in_place else i32([7] * batch, dev)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    flat = [torch.tensor([x for t in xs for x in t], dtype=torch.int64, device=dev) for xs in (drafts, targets)]
    ops.accept_tree(ops.make_pool(k, v), ops.make_tables(table.to(dev), i32(rows, dev)), i32([p for t in trees for p in t], dev),
                    i32(cu, dev), flat[0], flat[1], kn, vn, lens, counts, path, tokens, lengths_out=out, status=status)
    ops.raise_device_errors(status)
    paths = [accept(t, a, g, width) if r >= 0 else [] for t, a, g, r in zip(trees, drafts, targets, rows)]
    assert counts.tolist() == [len(p) for p in paths]
    assert path.tolist() == [p + [-1] * (width - len(p)) for p in paths]
    assert tokens.tolist() == [[g[i] for i in p] + [-1] * (width - len(p)) for p, g in zip(paths, targets)]
    assert (lens if in_place else out).tolist() == [c + len(p) for c, p in zip(ctx, paths)]
    assert in_place or lens.tolist() == ctx
    for b, p in enumerate(paths):
        for i, node in enumerate(p):
            blk, off = int(table[rows[b], (ctx[b] + i) // bs]), (ctx[b] + i) % bs
            want_k[:, blk, :, off] = kn[:, cu[b] + node]
            want_v[:, blk, :, off] = vn[:, cu[b] + node]
    assert torch.equal(k, want_k) and torch.equal(v, want_v)


def test_acceptance_without_a_block_is_reported(dev):
    from mini_inference_b200 import ops

    k = torch.zeros(1, 3, 1, 16, 64, dtype=torch.float16, device=dev)
    v = torch.zeros_like(k)
    ones = torch.ones(1, 2, 1, 64, dtype=torch.float16, device=dev)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    tok = torch.zeros(2, dtype=torch.int64, device=dev)
    outs = i32([0], dev), torch.zeros(1, 4, dtype=torch.int32, device=dev), torch.zeros(1, 4, dtype=torch.int64, device=dev)
    for table, length in (([[1]], 15), ([[1, -1]], 15), ([[1, 9]], 15)):
        ops.accept_tree(ops.make_pool(k, v), ops.make_tables(i32(table, dev)), i32([-1, 0], dev), i32([0, 2], dev), tok, tok, ones,
                        ones, i32([length], dev), *outs, status=status)
        with pytest.raises(IndexError):
            ops.raise_device_errors(status)
        assert (k[0, 1, 0, 15] == 1).all() and k.sum() == 64 and outs[0].item() == 2


def test_refusals(dev):
    from mini_inference_b200 import PkvError, ops

    one, two = i32([1], dev), i32([0, 1], dev)
    t = ops.make_tables(i32([[1]], dev))
    with pytest.raises(ValueError):
        ops.extend_tables(t, one, one.long(), one, one, one, 16, two, one)
    with pytest.raises(ValueError):
        ops.extend_tables(t, one, one, one, one, one, 16, one, one)  # cu_seqlens one short
    with pytest.raises(PkvError):
        ops.extend_tables(t, two, two, two, one, one, 16, i32([0] * 3, dev), two)  # a table of one row
    many = i32([0] * 4097, dev)
    with pytest.raises(PkvError):
        ops.extend_tables(ops.make_tables(i32([[1]] * 4097, dev)), many, many, many, one, one, 16, i32([0] * 4098, dev), many)
    m64 = torch.zeros(1, 9, dtype=torch.int64, device=dev)
    with pytest.raises(PkvError):
        ops.build_tree_metadata(one, two, one, m64, torch.zeros(1, dtype=torch.int64, device=dev))  # 9 words
    with pytest.raises(ValueError):
        ops.build_tree_metadata(one, two, one, m64[:, :1], torch.zeros(2, dtype=torch.int64, device=dev))
    k = torch.zeros(1, 2, 1, 16, 64, dtype=torch.float16, device=dev)
    pool = ops.make_pool(k, k.clone())
    tok, nodes = torch.zeros(1, dtype=torch.int64, device=dev), torch.zeros(1, 1, 1, 64, dtype=torch.float16, device=dev)
    path, tokens = torch.zeros(1, 65, dtype=torch.int32, device=dev), torch.zeros(1, 65, dtype=torch.int64, device=dev)
    with pytest.raises(PkvError):
        ops.accept_tree(pool, t, one, two, tok, tok, nodes, nodes, one, one.clone(), path, tokens)  # width 65
    with pytest.raises(ValueError):
        ops.accept_tree(pool, t, one, two, tok, tok, nodes.bfloat16().float(), nodes, one, one.clone(), path, tokens[:, :3])
