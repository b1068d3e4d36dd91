"""The operators of a speculative decoding step, in plain form and as this package runs them.

A serving step that verifies drafted tokens goes through five operators: block tables and slot
maps grown on the GPU from request lengths, the drafted trees' positions and ancestor masks,
rotary positions of the new rows, attention of a tree of drafted tokens over the paged cache,
and the greedy acceptance of a path with its K/V written to the cache. ``listed`` and ``draw``
give cases, ``prepare`` their inputs, ``run`` one pass, ``work`` what a pass has to move and
compute, and ``exact`` the computed outputs from their definitions in 64 bits.

Block size 16 throughout; head shapes are those of the two model families of this package
(14 / 2 heads of 64 and 28 / 4 heads of 128) and generic ones.
"""

import math

import numpy as np
import torch

own = False

BS = 16
SHAPES = {"14/2/64": (14, 2, 64), "28/4/128": (28, 4, 128), "8/8/64": (8, 8, 64), "12/4/64": (12, 4, 64),
          "16/1/128": (16, 1, 128), "32/8/128": (32, 8, 128)}
DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16}


# ---------------------------------------------------------------- cases

def listed():
    return [
        # One user's request early in its answer: a small drafted tree, where launch latency counts.
        dict(name="attention, one request", op="attention", shape="14/2/64", dtype="float16", batch=1, ctx_lo=129,
             ctx_hi=129, nodes_lo=8, nodes_hi=8, branch=2),
        # A serving batch of the smaller model: ragged contexts and trees, one drafted token to 26.
        dict(name="attention, serving batch", op="attention", shape="14/2/64", dtype="float16", batch=64, ctx_lo=128,
             ctx_hi=2048, nodes_lo=1, nodes_hi=26, branch=3),
        # Long documents on the larger model's heads: the cache is streamed once for every tree.
        dict(name="attention, long contexts", op="attention", shape="28/4/128", dtype="bfloat16", batch=16,
             ctx_lo=8191, ctx_hi=32001, nodes_lo=9, nodes_hi=18, branch=2),
        # Few requests with wide trees: many rows for each cached key.
        dict(name="attention, wide trees", op="attention", shape="28/4/128", dtype="bfloat16", batch=4, ctx_lo=1000,
             ctx_hi=4100, nodes_lo=129, nodes_hi=256, branch=4),
        # A decode batch of a model that rotates the first half of each head, pairs interleaved.
        dict(name="rotary, decode batch", op="rotary", shape="28/4/128", dtype="float16", rows=64, rotary=64,
             interleaved=True, factor=1.0, far=131072, append=False),
        # A packed prefill stretched past its trained length, appended to the cache as it is rotated.
        dict(name="rotary, packed prefill", op="rotary", shape="28/4/128", dtype="bfloat16", rows=8192, rotary=128,
             interleaved=False, factor=4.0, far=131072, append=True),
        # One new token for each of a serving batch's requests.
        dict(name="tables, decode batch", op="tables", batch=250, new_lo=1, new_hi=1, len_lo=0, len_hi=2047),
        # Chunks of long prompts beside short ones, a whole step's token budget.
        dict(name="tables, prompt chunks", op="tables", batch=61, new_lo=1, new_hi=4096, len_lo=0, len_hi=30000),
        # One small drafted tree.
        dict(name="tree, one request", op="tree", batch=1, nodes_lo=8, nodes_hi=8, branch=2),
        # A full serving batch of trees of up to 256 drafted tokens.
        dict(name="tree, serving batch", op="tree", batch=256, nodes_lo=64, nodes_hi=256, branch=3),
        # The accepted path of one request, all layers of the smaller model.
        dict(name="accept, one request", op="accept", shape="14/2/64", dtype="float16", batch=1, layers=24, nodes_lo=8,
             nodes_hi=8, branch=2),
        # A serving batch's accepted paths, all layers of the larger model.
        dict(name="accept, serving batch", op="accept", shape="28/4/128", dtype="bfloat16", batch=128, layers=28,
             nodes_lo=16, nodes_hi=40, branch=2),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _drawn(rng, op):
    shape, dtype = rng.choice(sorted(SHAPES)), rng.choice(sorted(DTYPES))
    if op == "attention":
        nodes = _log(rng, 1, 256)
        ctx = _log(rng, 1, 32000)
        return dict(op=op, shape=shape, dtype=dtype, batch=_log(rng, 1, 64), ctx_lo=rng.choice([0, ctx // 3, ctx]),
                    ctx_hi=ctx, nodes_lo=rng.choice([1, nodes]), nodes_hi=nodes, branch=rng.randint(1, 4))
    if op == "rotary":
        d = SHAPES[shape][2]
        return dict(op=op, shape=shape, dtype=dtype, rows=_log(rng, 1, 8192), rotary=rng.choice([d, d // 2, d // 4]),
                    interleaved=rng.random() < 0.5, factor=rng.choice([1.0, 2.0, 8.0]), far=_log(rng, 16, 1000000),
                    append=rng.random() < 0.5)
    if op == "tables":
        new, length = _log(rng, 1, 4096), _log(rng, 1, 30000)
        return dict(op=op, batch=_log(rng, 1, 1000), new_lo=rng.choice([0, 1, new]), new_hi=new,
                    len_lo=rng.choice([0, length]), len_hi=length)
    nodes = _log(rng, 1, 256 if op == "tree" else 64)
    case = dict(op=op, batch=_log(rng, 1, 256), nodes_lo=rng.choice([1, nodes]), nodes_hi=nodes,
                branch=rng.randint(1, 4))
    if op == "accept":
        case |= dict(shape=shape, dtype=dtype, layers=_log(rng, 1, 28))
    return case


def _cost(case):
    w = work(case)
    return w["bytes"] + w["flops"] / 200


def draw(rng):
    op = rng.choice(["attention", "attention", "rotary", "tables", "tree", "accept"])
    most = max(_cost(c) for c in listed() if c["op"] == op)
    case = _drawn(rng, op)
    while _cost(case) > most or (op == "attention" and case["batch"] * case["ctx_hi"] > 16 * 32001):
        case = _drawn(rng, op)
    return case


# ---------------------------------------------------------------- inputs

def _spread(lo, hi, n):
    """n whole numbers evenly over lo..hi (the sum does not depend on a seed)."""
    return np.rint(np.linspace(lo, hi, n)).astype(np.int64) if n > 1 else np.array([hi])


def _parents(counts, branch):
    """Trees in breadth-first order: node i hangs below (i - 1) // branch; -1 for the root."""
    return np.concatenate([np.where(np.arange(n) > 0, (np.arange(n) - 1) // branch, -1) for n in counts])


def _gpu(a, dtype):
    return torch.from_numpy(np.ascontiguousarray(a)).to("cuda", dtype)


def _trees(case, rng):
    counts = rng.permutation(_spread(case["nodes_lo"], case["nodes_hi"], case["batch"]))
    cu = np.concatenate([[0], np.cumsum(counts)])
    return counts, cu, _parents(counts, case["branch"])


def _depths(parents, counts):
    out, base = np.zeros(len(parents), np.int64), 0
    for n in counts:
        for i in range(1, n):
            out[base + i] = out[base + parents[base + i]] + 1
        base += n
    return out


def _masks(parents, counts, words):
    """Each node's ancestors and itself as bits, 64 nodes to a word."""
    out, base = np.zeros((len(parents), words), np.uint64), 0
    for n in counts:
        for i in range(n):
            if i:
                out[base + i] = out[base + parents[base + i]]
            out[base + i, i // 64] |= np.uint64(1) << np.uint64(i % 64)
        base += n
    return out.view(np.int64)


def _pools(case, layers, blocks, gen):
    _, hkv, d = SHAPES[case["shape"]]
    k = torch.empty(layers, blocks + 1, hkv, BS, d, dtype=DTYPES[case["dtype"]], device="cuda")
    v = torch.empty_like(k)
    return k.normal_(generator=gen), v.normal_(generator=gen)


def _tables(lengths, rng):
    """Block tables that hold `lengths` tokens, blocks in no order; -1 past a request's blocks."""
    need = -(-lengths // BS)
    total, cols = int(need.sum()), max(1, int(need.max()))
    order, t = rng.permutation(total), np.full((len(lengths), cols), -1, np.int64)
    t[np.arange(cols)[None, :] < need[:, None]] = order
    return t, total


def _frequencies(case):
    """theta^(-2 i / rotary), slow pairs slowed further by `factor` (a linear ramp over the pairs between)."""
    half = case["rotary"] // 2
    i = np.arange(half, dtype=np.float64)
    f = 1e6 ** (-i / half)
    ramp = np.clip((i - half / 8) / (half / 2), 0, 1) if case["factor"] > 1 else np.zeros(half)
    return f * (1 - ramp) + f / case["factor"] * ramp, 0.1 * math.log(case["factor"]) + 1.0


def prepare(case, seed):
    rng = np.random.RandomState(seed % (1 << 31))
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = PREPARE[case["op"]](case, rng, gen)
    s["op"] = case["op"]
    if own:  # the handles that a program keeps: how the package sees the same pool and tables, and a workspace
        from mini_inference_b200 import ops
        if "pool_k" in s:
            s["pool"] = ops.make_pool(s["pool_k"], s["pool_v"])
        if "tables" in s:
            s["handle"] = ops.make_tables(s["tables"])
        if case["op"] == "attention":
            s["workspace"] = ops.tree_attention_workspace(s["pool"], case["batch"], "cuda")
    return s


def _prepare_attention(case, rng, gen):
    hq, hkv, d = SHAPES[case["shape"]]
    dtype = DTYPES[case["dtype"]]
    counts, cu, parents = _trees(case, rng)
    ctx = rng.permutation(_spread(case["ctx_lo"], case["ctx_hi"], case["batch"]))
    table, blocks = _tables(ctx, rng)
    pool_k, pool_v = _pools(case, 1, blocks, gen)
    n = int(cu[-1])
    # One projection's rows: the nodes' keys stand alone (they are rotated), their values are a view.
    qkv = torch.empty(n, (hq + 2 * hkv) * d, dtype=dtype, device="cuda").normal_(generator=gen)
    q = torch.empty(n, hq, d, dtype=dtype, device="cuda").normal_(generator=gen)
    k = torch.empty(n, hkv, d, dtype=dtype, device="cuda").normal_(generator=gen)
    words = -(-case["nodes_hi"] // 64)
    return dict(pool_k=pool_k, pool_v=pool_v, tables=_gpu(table, torch.int32), q=q, k_nodes=k,
                v_nodes=qkv[:, (hq + hkv) * d:].view(n, hkv, d), cu_nodes=_gpu(cu, torch.int32),
                context_lens=_gpu(ctx, torch.int32), mask=_gpu(_masks(parents, counts, words), torch.int64),
                max_nodes=case["nodes_hi"], max_ctx=case["ctx_hi"])


def _prepare_rotary(case, rng, gen):
    hq, hkv, d = SHAPES[case["shape"]]
    n = case["rows"]
    freq, factor = _frequencies(case)
    qkv = torch.empty(n, (hq + 2 * hkv) * d, dtype=DTYPES[case["dtype"]], device="cuda").normal_(generator=gen)
    blocks = -(-n // BS) if case["append"] else 1
    pool_k, pool_v = _pools(case, 1, blocks, gen)
    return dict(pool_k=pool_k, pool_v=pool_v, qkv=qkv, hq=hq, interleaved=case["interleaved"], factor=factor,
                positions=_gpu(rng.randint(0, case["far"], n), torch.int64), freq=_gpu(freq, torch.float64),
                slots=_gpu(rng.permutation(blocks * BS)[:n], torch.int64) if case["append"] else None)


def _prepare_tables(case, rng, gen):
    b = case["batch"]
    new = rng.permutation(_spread(case["new_lo"], case["new_hi"], b))
    length = rng.permutation(_spread(case["len_lo"], case["len_hi"], b))
    held = -(-length // BS)
    cols = -(-(case["len_hi"] + case["new_hi"]) // BS) + 3
    fresh = int((-(-(length + new) // BS)).sum() - held.sum())
    order = rng.permutation(int(held.sum()) + fresh + 5)
    table = np.full((b, cols), -1, np.int64)
    table[np.arange(cols)[None, :] < held[:, None]] = order[:int(held.sum())]
    s = dict(tables=_gpu(table, torch.int32), lengths=_gpu(length, torch.int32), new=_gpu(new, torch.int32),
             held=_gpu(held, torch.int32), free=_gpu(np.concatenate([[0, 0], order[int(held.sum()):]]), torch.int32),
             head=_gpu([2], torch.int32), total=int(new.sum()))
    i32, i64 = dict(dtype=torch.int32, device="cuda"), dict(dtype=torch.int64, device="cuda")
    return s | dict(cu=torch.empty(b + 1, **i32), ctx=torch.empty(b, **i32), positions=torch.empty(s["total"], **i64),
                    slots=torch.empty(s["total"], **i64), held_out=torch.empty(b, **i32), head_out=torch.empty(1, **i32))


def _prepare_tree(case, rng, gen):
    counts, cu, parents = _trees(case, rng)
    n, words = int(cu[-1]), -(-case["nodes_hi"] // 64)
    return dict(parents=_gpu(parents, torch.int32), cu_nodes=_gpu(cu, torch.int32), max_nodes=case["nodes_hi"],
                context_lens=_gpu(rng.randint(0, 30000, case["batch"]), torch.int32),
                mask=torch.empty(n, words, dtype=torch.int64, device="cuda"),
                positions=torch.empty(n, dtype=torch.int64, device="cuda"))


def _chain(case, n):
    """Nodes on the way down from the root by the last child, while there is one."""
    path, i = [0], 0
    while case["branch"] * i + 1 < n:
        i = min(case["branch"] * (i + 1), n - 1)
        path.append(i)
    return path


def _accepted(case):
    """How many nodes each tree's path has, in the order of the trees' sizes (no seed in it)."""
    counts = _spread(case["nodes_lo"], case["nodes_hi"], case["batch"])
    return [min(len(_chain(case, int(n))), 1 + (5 * b + 3) % 6) for b, n in enumerate(counts)]


def _prepare_accept(case, rng, gen):
    _, hkv, d = SHAPES[case["shape"]]
    b, dtype = case["batch"], DTYPES[case["dtype"]]
    sizes, lens = _spread(case["nodes_lo"], case["nodes_hi"], b), _accepted(case)
    order = rng.permutation(b)
    counts = sizes[order]
    cu = np.concatenate([[0], np.cumsum(counts)])
    n = int(cu[-1])
    draft, target = rng.randint(0, 30000, n), rng.randint(30000, 150000, n)
    for i, j in enumerate(order):  # the target model's answers along the path; elsewhere it disagrees
        path = cu[i] + np.array(_chain(case, int(counts[i]))[:lens[j]])
        target[path[:-1]] = draft[path[1:]]
    ctx = rng.permutation(_spread(0, 200, b))
    table, blocks = _tables(ctx + case["nodes_hi"], rng)
    pool_k, pool_v = _pools(case, case["layers"], blocks, gen)
    k = torch.empty(case["layers"], n, hkv, d, dtype=dtype, device="cuda").normal_(generator=gen)
    v = torch.empty_like(k).normal_(generator=gen)
    width = 8
    return dict(pool_k=pool_k, pool_v=pool_v, tables=_gpu(table, torch.int32), k_nodes=k, v_nodes=v,
                parents=_gpu(_parents(counts, case["branch"]), torch.int32), cu_nodes=_gpu(cu, torch.int32),
                draft=_gpu(draft, torch.int64), target=_gpu(target, torch.int64), context_lens=_gpu(ctx, torch.int32),
                counts=torch.empty(b, dtype=torch.int32, device="cuda"), max_nodes=case["nodes_hi"], width=width,
                path=torch.empty(b, width, dtype=torch.int32, device="cuda"),
                tokens=torch.empty(b, width, dtype=torch.int64, device="cuda"),
                lengths_out=torch.empty(b, dtype=torch.int32, device="cuda"))


PREPARE = {"attention": _prepare_attention, "rotary": _prepare_rotary, "tables": _prepare_tables,
                   "tree": _prepare_tree, "accept": _prepare_accept}


# ---------------------------------------------------------------- one pass

def run(s):
    if own:
        return OWN[s["op"]](s)
    return PLAIN[s["op"]](s)


def _own_attention(s):
    from mini_inference_b200 import ops
    return ops.tree_attention(s["pool"], 0, s["handle"], s["q"], s["k_nodes"], s["v_nodes"], s["cu_nodes"],
                              s["context_lens"], s["mask"], s["max_nodes"], s["workspace"])


def _own_rotary(s):
    from mini_inference_b200 import ops
    if s["slots"] is not None:
        q, _, _ = ops.rotary_append(s["pool"], 0, s["qkv"], s["positions"], s["freq"], s["hq"],
                                    interleaved=s["interleaved"], attention_factor=s["factor"],
                                    slot_mapping=s["slots"])
        return q, s["pool_k"], s["pool_v"]
    return ops.rotary_append(s["pool"], 0, s["qkv"], s["positions"], s["freq"], s["hq"], interleaved=s["interleaved"],
                             attention_factor=s["factor"], k_out=True, v_out=True)


def _own_tables(s):
    from mini_inference_b200 import ops
    ops.extend_tables(s["handle"], s["lengths"], s["new"], s["held"], s["free"], s["head"], BS, s["cu"], s["ctx"],
                      s["positions"], s["slots"], held_out=s["held_out"], free_head_out=s["head_out"])
    return {k: s[k] for k in ("tables", "cu", "ctx", "positions", "slots", "held_out", "head_out")}


def _own_tree(s):
    from mini_inference_b200 import ops
    ops.build_tree_metadata(s["parents"], s["cu_nodes"], s["context_lens"], s["mask"], s["positions"])
    return s["mask"], s["positions"]


def _own_accept(s):
    from mini_inference_b200 import ops
    ops.accept_tree(s["pool"], s["handle"], s["parents"], s["cu_nodes"], s["draft"], s["target"], s["k_nodes"],
                    s["v_nodes"], s["context_lens"], s["counts"], s["path"], s["tokens"], lengths_out=s["lengths_out"])
    return {k: s[k] for k in ("counts", "path", "tokens", "lengths_out", "pool_k", "pool_v")}


OWN = {"attention": _own_attention, "rotary": _own_rotary, "tables": _own_tables, "tree": _own_tree,
       "accept": _own_accept}


def _padded(s, most):
    """For trees packed end to end: each tree's rows as [batch, most], and which of them there are."""
    cu = s["cu_nodes"].long()
    at = torch.arange(most, device="cuda")
    there = at < (cu[1:] - cu[:-1])[:, None]
    return torch.where(there, cu[:-1, None] + at, 0), there


def _plain_attention(s):
    rows, there = _padded(s, s["max_nodes"])
    b, t = rows.shape
    q, kn, vn = (s[x][rows].float() for x in ("q", "k_nodes", "v_nodes"))
    hq, hkv, d = q.shape[2], kn.shape[2], q.shape[3]
    blocks = s["tables"][:, :-(-s["max_ctx"] // BS)].long().clamp(min=0)
    ctx = s["context_lens"].long()
    seen = torch.arange(blocks.shape[1] * BS, device="cuda") < ctx[:, None]  # [b, keys]
    k = torch.cat([s["pool_k"][0][blocks].float().transpose(1, 2).reshape(b, hkv, -1, d), kn.transpose(1, 2)], 2)
    v = torch.cat([s["pool_v"][0][blocks].float().transpose(1, 2).reshape(b, hkv, -1, d), vn.transpose(1, 2)], 2)
    at = torch.arange(t, device="cuda")
    tree = (s["mask"][rows][:, :, at // 64] >> (at % 64)) & 1
    allowed = torch.cat([seen[:, None, :].expand(-1, t, -1), (tree > 0) & there[:, None, :]], 2)
    x = q.view(b, t, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, -1, d) @ k.transpose(2, 3) / math.sqrt(d)
    x = x.view(b, hkv, hq // hkv, t, -1).masked_fill(~allowed[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = (p.reshape(b, hkv, -1, p.shape[-1]) @ v).view(b, hkv, hq // hkv, t, d) / torch.where(total > 0, total, 1.0)
    return o.permute(0, 3, 1, 2, 4).reshape(b, t, hq, d)[there].to(s["q"].dtype)


def _plain_rotary(s):
    n = s["qkv"].shape[0]
    hkv, d = s["pool_k"].shape[2], s["pool_k"].shape[4]
    r = 2 * s["freq"].numel()
    angle = s["positions"].double()[:, None] * s["freq"]
    cos, sin = ((f(angle) * s["factor"]).float()[:, None, :] for f in (torch.cos, torch.sin))
    x = s["qkv"].view(n, -1, d)
    heads = x[:, :s["hq"] + hkv, :r].float()
    if s["interleaved"]:
        a, b = heads[..., 0::2], heads[..., 1::2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = heads[..., :r // 2], heads[..., r // 2:]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    y = torch.cat([y.to(x.dtype), x[:, :s["hq"] + hkv, r:]], -1)
    q, k, v = y[:, :s["hq"]], y[:, s["hq"]:], x[:, s["hq"] + hkv:]
    if s["slots"] is None:
        return q.contiguous(), k.contiguous(), v.contiguous()
    s["pool_k"][0, s["slots"] // BS, :, s["slots"] % BS] = k
    s["pool_v"][0, s["slots"] // BS, :, s["slots"] % BS] = v
    return q.contiguous(), s["pool_k"], s["pool_v"]


def _plain_tables(s):
    length, new, held = s["lengths"].long(), s["new"].long(), s["held"].long()
    need = torch.maximum(torch.div(length + new + BS - 1, BS, rounding_mode="floor"), held)
    fresh = need - held
    first = fresh.cumsum(0) - fresh
    head = s["head"].long()
    col = torch.arange(s["tables"].shape[1], device="cuda")
    grown = (col >= held[:, None]) & (col < need[:, None])
    take = torch.where(grown, head + first[:, None] + col - held[:, None], 0)
    s["tables"].copy_(torch.where(grown, s["free"][take], s["tables"]))
    cu = torch.cat([new.new_zeros(1), new.cumsum(0)])
    token = torch.arange(s["total"], device="cuda")
    of = torch.searchsorted(cu, token, right=True) - 1
    pos = length[of] + token - cu[of]
    slot = s["tables"][of, pos // BS].long() * BS + pos % BS
    return dict(tables=s["tables"], cu=cu.int(), ctx=(length + new).int(), positions=pos, slots=slot, held_out=need.int(),
                head_out=(head + fresh.sum()).int())


def _plain_tree(s):
    rows, there = _padded(s, s["max_nodes"])
    b, t = rows.shape
    at = torch.arange(t, device="cuda")
    parent = torch.where(there, s["parents"][rows].long(), -1)
    below = (parent[:, :, None] == at).double()  # [b, node, parent]
    reach = below + torch.eye(t, device="cuda", dtype=torch.double)
    # Ancestors by repeated squaring: 2^8 steps up cover every tree of up to 256 nodes.
    for _ in range(max(1, (t - 1).bit_length())):
        reach = (reach @ reach > 0).double()
    bits = reach.bool() & there[:, :, None]
    words = s["mask"].shape[1]
    pad = torch.zeros(b, t, 64 * words, dtype=torch.int64, device="cuda")
    pad[:, :, :t] = bits.long() << (at % 64)
    mask = pad.view(b, t, words, 64).sum(-1)
    pos = s["context_lens"].long()[:, None] + bits.sum(-1) - 1
    return mask[there], pos[there]


def _plain_accept(s):
    rows, there = _padded(s, s["max_nodes"])
    b, t = rows.shape
    at = torch.arange(t, device="cuda")
    parent = torch.where(there, s["parents"][rows].long(), -1)
    draft, target = s["draft"][rows], s["target"][rows]
    agrees = (parent >= 0) & (draft == target.gather(1, parent.clamp(min=0)))
    twin = (parent[:, :, None] == parent[:, None, :]) & agrees[:, :, None] & agrees[:, None, :] & (at < at[:, None])
    good = (agrees & ~twin.any(2)) | (there & (at == 0))
    reach = ((parent[:, :, None] == at).double() + torch.eye(t, device="cuda", dtype=torch.double))
    for _ in range(max(1, (t - 1).bit_length())):
        reach = (reach @ reach > 0).double()
    whole = good & ~((reach > 0) & ~good[:, None, :]).any(2)
    place = whole.long().cumsum(1) - 1  # a path's nodes stand in the order of their indexes
    whole &= place < s["width"]
    count = whole.sum(1)
    seq, node = whole.nonzero(as_tuple=True)
    path = torch.full((b, s["width"]), -1, dtype=torch.int32, device="cuda")
    tokens = torch.full((b, s["width"]), -1, dtype=torch.int64, device="cuda")
    at_place = place[seq, node]
    path[seq, at_place] = node.int()
    tokens[seq, at_place] = target[seq, node]
    pos = s["context_lens"].long()[seq] + at_place
    block = s["tables"][seq, pos // BS].long()
    src = rows[seq, node]
    s["pool_k"][:, block, :, pos % BS] = s["k_nodes"][:, src].transpose(0, 1)
    s["pool_v"][:, block, :, pos % BS] = s["v_nodes"][:, src].transpose(0, 1)
    return dict(counts=count.int(), path=path, tokens=tokens, lengths_out=s["context_lens"] + count.int(),
                pool_k=s["pool_k"], pool_v=s["pool_v"])


PLAIN = {"attention": _plain_attention, "rotary": _plain_rotary, "tables": _plain_tables, "tree": _plain_tree,
         "accept": _plain_accept}


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    op, b = case["op"], case.get("batch", 0)
    if op == "rotary":
        hq, hkv, d = SHAPES[case["shape"]]
        n = case["rows"]
        return {"bytes": n * (2 * (hq + 2 * hkv) * d * 2 + 8 + (8 if case["append"] else 0)) + 4 * case["rotary"],
                "flops": n * 3 * (hq + hkv) * case["rotary"]}
    if op == "tables":
        new, length = _spread(case["new_lo"], case["new_hi"], b), _spread(case["len_lo"], case["len_hi"], b)
        tokens = int(new.sum())
        # Four numbers read and three written for a request; a block table entry for each 16
        # tokens (read, or taken from the free list and written), position and slot of each.
        return {"bytes": b * 28 + tokens * 16 + 8 * (tokens // BS + b), "flops": 2 * tokens}
    nodes = int(_spread(case["nodes_lo"], case["nodes_hi"], b).sum())
    words = -(-case["nodes_hi"] // 64)
    if op == "tree":
        return {"bytes": nodes * (4 + 8 + 8 * words) + 8 * b, "flops": nodes * 8}
    hq, hkv, d = SHAPES[case["shape"]]
    if op == "accept":
        moved = sum(_accepted(case)) * case["layers"] * 2 * hkv * d * 2
        return {"bytes": 2 * moved + nodes * 20 + b * 8 * 13, "flops": nodes * 4}
    counts = _spread(case["nodes_lo"], case["nodes_hi"], b)
    ctx = _spread(case["ctx_lo"], case["ctx_hi"], b)
    keys = int(ctx.sum())
    scores = int(counts.mean() * keys) + int((counts * counts).sum())  # seeds pair contexts and trees anew
    return {"bytes": (keys + nodes) * hkv * d * 4 + nodes * (hq * d * 4 + 8 * words) + 4 * (keys // BS + b),
            "flops": 4 * scores * hq * d}


# ---------------------------------------------------------------- from the definitions, in 64 bits

def exact(case, seed):
    if case["op"] == "attention":
        return _exact_attention(prepare(case, seed))
    if case["op"] == "rotary":
        return _exact_rotary(prepare(case, seed))
    return None  # whole numbers and moved rows: nothing is computed


def _exact_attention(s):
    cu, ctx = s["cu_nodes"].tolist(), s["context_lens"].tolist()
    hq, hkv, d = s["q"].shape[1], s["k_nodes"].shape[1], s["q"].shape[2]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, (lo, hi) in enumerate(zip(cu, cu[1:])):
        block = s["tables"][b, :-(-ctx[b] // BS)].long()
        bits = s["mask"][lo:hi].cpu().numpy().view(np.uint64)
        vis = np.array([[bool(int(w[j // 64]) >> (j % 64) & 1) for j in range(hi - lo)] for w in bits])
        vis = torch.from_numpy(np.concatenate([np.ones((hi - lo, ctx[b]), bool), vis], 1)).cuda()
        for h in range(hkv):
            k = torch.cat([s["pool_k"][0, block, h].reshape(-1, d)[:ctx[b]], s["k_nodes"][lo:hi, h]]).double()
            v = torch.cat([s["pool_v"][0, block, h].reshape(-1, d)[:ctx[b]], s["v_nodes"][lo:hi, h]]).double()
            for g in range(h * hq // hkv, (h + 1) * hq // hkv):
                x = s["q"][lo:hi, g].double() @ k.T * d ** -0.5
                x[~vis] = -math.inf
                out[lo:hi, g] = torch.nan_to_num(torch.softmax(x, -1), nan=0.0) @ v
    return out


def _exact_rotary(s):
    n, hkv, d = s["qkv"].shape[0], s["pool_k"].shape[2], s["pool_k"].shape[4]
    half = s["freq"].numel()
    z = torch.polar(torch.full((), float(s["factor"]), dtype=torch.float64, device="cuda"),
                    s["positions"].double()[:, None] * s["freq"])[:, None, :]
    x = s["qkv"].double().view(n, -1, d)
    y = x.clone()
    turned = slice(0, s["hq"] + hkv)
    if s["interleaved"]:
        pair = torch.view_as_complex(x[:, turned, :2 * half].reshape(n, -1, half, 2).contiguous()) * z
        y[:, turned, :2 * half] = torch.view_as_real(pair).flatten(-2)
    else:
        pair = torch.complex(x[:, turned, :half].contiguous(), x[:, turned, half:2 * half].contiguous()) * z
        y[:, turned, :half], y[:, turned, half:2 * half] = pair.real, pair.imag
    q, k, v = y[:, :s["hq"]], y[:, s["hq"]:s["hq"] + hkv], y[:, s["hq"] + hkv:]
    if s["slots"] is None:
        return q, k, v
    pk, pv = s["pool_k"].double(), s["pool_v"].double()
    pk[0, s["slots"] // BS, :, s["slots"] % BS] = k
    pv[0, s["slots"] // BS, :, s["slots"] % BS] = v
    return q, pk, pv
