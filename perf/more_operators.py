"""Operators of a decoder layer with query/key norms, positions on several axes and experts.

A prompt that holds images or video beside text places each token on three axes (time, height,
width); queries and keys are normalised head by head and rotated by those positions as they are
appended to the paged cache; and the MLP is a mixture of experts. Three operators: ``positions``
(the axes' positions from the prompt's media), ``rotary`` (norm, rotation, append) and
``experts`` (router and experts' products). ``listed`` and ``draw`` give cases, ``prepare``
their inputs, ``run`` one pass, ``work`` what a pass has to move and compute, and ``exact`` the
computed outputs from their definitions in 64 bits.

Block size 16 throughout; head shapes are those of the two model families of this package
(14 / 2 heads of 64 and 28 / 4 heads of 128) and generic ones.
"""

import math

import numpy as np
import torch

own = False

BS = 16
EPS = 1e-6
SHAPES = {"14/2/64": (14, 2, 64), "28/4/128": (28, 4, 128), "8/8/64": (8, 8, 64), "16/1/128": (16, 1, 128),
          "32/8/128": (32, 8, 128), "8/2/256": (8, 2, 256)}
DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16}
OPS = ("positions", "rotary", "experts")


# ---------------------------------------------------------------- cases

def listed():
    return [
        # One new token for each of a serving batch's conversations, each with a few images behind it.
        dict(name="positions, decode batch", op="positions", batch=64, new_lo=1, new_hi=1, behind=1500, spans=4, side=24),
        # A step's budget of prompts, most of their tokens images and clips.
        dict(name="positions, packed prompts", op="positions", batch=9, new_lo=1200, new_hi=6000, behind=0, spans=12, side=28),
        # One user's token on the larger model's heads: launch latency.
        dict(name="rotary, one token", op="rotary", shape="28/4/128", dtype="bfloat16", rows=1, rotary=128, axes=3,
             interleaved=False, norm=True, far=32768, append=False),
        # A decode batch of the smaller model, all axes alike.
        dict(name="rotary, decode batch", op="rotary", shape="14/2/64", dtype="float16", rows=64, rotary=64, axes=1,
             interleaved=False, norm=True, far=32768, append=False),
        # A chunk of an odd length, half of each head rotated, pairs side by side.
        dict(name="rotary, odd chunk", op="rotary", shape="32/8/128", dtype="float16", rows=1013, rotary=64, axes=1,
             interleaved=True, norm=True, far=131072, append=True),
        # Packed prompts with images, appended to the cache as they are rotated.
        dict(name="rotary, packed prompts", op="rotary", shape="28/4/128", dtype="bfloat16", rows=8192, rotary=128, axes=3,
             interleaved=False, norm=True, far=131072, append=True),
        # One user's token through many small experts: the touched weights and the latency of the chain.
        dict(name="experts, one token", op="experts", dtype="bfloat16", tokens=1, hidden=2048, inter=768, experts=64, top=8),
        # A few tokens (a small drafted tree) on the smaller model's width.
        dict(name="experts, few tokens", op="experts", dtype="float16", tokens=7, hidden=896, inter=1216, experts=32, top=4),
        # A few requests through large experts of the larger model's width.
        dict(name="experts, large experts", op="experts", dtype="bfloat16", tokens=16, hidden=3584, inter=2368, experts=16,
             top=2),
        # A serving batch: every expert is touched, each by few tokens.
        dict(name="experts, decode batch", op="experts", dtype="bfloat16", tokens=64, hidden=2048, inter=1024, experts=64,
             top=8),
        # Drafted trees of a serving batch: odd numbers throughout.
        dict(name="experts, drafted trees", op="experts", dtype="float16", tokens=333, hidden=896, inter=616, experts=60,
             top=4),
        # A packed prefill.
        dict(name="experts, packed prompts", op="experts", dtype="bfloat16", tokens=2048, hidden=2048, inter=768, experts=64,
             top=8),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _drawn(rng, op):
    dtype = rng.choice(sorted(DTYPES))
    if op == "positions":
        new = _log(rng, 1, 6000)
        return dict(op=op, batch=_log(rng, 1, 256), new_lo=rng.choice([1, new]), new_hi=new, behind=_log(rng, 1, 4000),
                    spans=_log(rng, 1, 40), side=_log(rng, 1, 40))
    if op == "rotary":
        shape = rng.choice(sorted(SHAPES))
        d = SHAPES[shape][2]
        return dict(op=op, shape=shape, dtype=dtype, rows=_log(rng, 1, 8192), rotary=rng.choice([d, d // 2, d // 4]),
                    axes=rng.choice([1, 2, 3]), interleaved=rng.random() < 0.3, norm=rng.random() < 0.8,
                    far=_log(rng, 16, 1000000), append=rng.random() < 0.5)
    experts = rng.choice([4, 8, 16, 32, 60, 64, 128])
    return dict(op=op, dtype=dtype, tokens=_log(rng, 1, 2048), hidden=rng.choice([512, 896, 1000, 2048, 3584]),
                inter=8 * _log(rng, 8, 300), experts=experts, top=rng.choice([1, 2, 4, 8][:3 if experts < 8 else 4]))


def _cost(case):
    w = work(case)
    return w["bytes"] + w["flops"] / 200


def draw(rng):
    op = rng.choice(["positions", "rotary", "rotary", "experts", "experts", "experts"])
    most = max(_cost(c) for c in listed() if c["op"] == op)
    case = _drawn(rng, op)
    while _cost(case) > most or (op == "experts" and case["experts"] * case["hidden"] * case["inter"] > 64 * 2048 * 1024):
        case = _drawn(rng, op)
    return case


# ---------------------------------------------------------------- inputs

def _spread(lo, hi, n):
    """n whole numbers evenly over lo..hi (the sum does not depend on a seed)."""
    return np.rint(np.linspace(lo, hi, n)).astype(np.int64) if n > 1 else np.array([hi])


def _gpu(a, dtype):
    return torch.from_numpy(np.ascontiguousarray(a)).to("cuda", dtype)


def prepare(case, seed):
    rng = np.random.RandomState(seed % (1 << 31))
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = PREPARE[case["op"]](case, rng, gen)
    s["op"] = case["op"]
    if own:  # the handles that a program keeps: how the package sees the pool, and a workspace
        from mini_inference_b200 import ops
        if "pool_k" in s:
            s["pool"] = ops.make_pool(s["pool_k"], s["pool_v"])
        if case["op"] == "experts":
            s["workspace"] = ops.expert_mlp_workspace(case["tokens"], case["experts"], case["top"], case["hidden"],
                                                      case["inter"], "cuda")
    return s


def _media(rng, length, spans, side):
    """Up to `spans` images and clips with text between them, within `length` tokens: (start, frames, height, width, step)."""
    rows, at = [], 0
    for _ in range(spans):
        at += int(rng.randint(0, 40))
        frames = int(rng.choice([1, 1, 1, 4]))
        h, w = int(rng.randint(1, side + 1)), int(rng.randint(1, side + 1))
        if at + frames * h * w > length:
            break
        rows.append((at, frames, h, w, int(rng.choice([1, 2])) if frames > 1 else 1))
        at += frames * h * w
    return rows


def _prepare_positions(case, rng, gen):
    b = case["batch"]
    new = rng.permutation(_spread(case["new_lo"], case["new_hi"], b))
    start = rng.permutation(_spread(case["behind"] // 2, case["behind"], b))
    slots = rng.permutation(b + 3)[:b]  # the sequences' rows of the media table
    media, counts = np.zeros((b + 3, case["spans"], 5), np.int64), np.zeros(b + 3, np.int64)
    for i in range(b):
        rows = _media(rng, int(start[i] + new[i]), case["spans"], case["side"])
        counts[slots[i]] = len(rows)
        if rows:
            media[slots[i], :len(rows)] = rows
    cu = np.concatenate([[0], np.cumsum(new)])
    pos = np.concatenate([np.arange(a, a + n) for a, n in zip(start, new)])
    return dict(positions=_gpu(pos, torch.int64), cu_seqlens=_gpu(cu, torch.int32), media=_gpu(media, torch.int32),
                media_counts=_gpu(counts, torch.int32), seq_rows=_gpu(slots, torch.int32),
                out=torch.empty(3, len(pos), dtype=torch.int64, device="cuda"))


def _pair_axes(half, axes):
    """Which axis turns each pair: a quarter of the pairs by the first, the rest by the others evenly."""
    first = half if axes == 1 else half // 4
    cuts = np.linspace(first, half, axes).round().astype(np.int64)
    return np.searchsorted(cuts, np.arange(half), side="right")


def _prepare_rotary(case, rng, gen):
    hq, hkv, d = SHAPES[case["shape"]]
    n, dtype = case["rows"], DTYPES[case["dtype"]]
    half = case["rotary"] // 2
    qkv = torch.empty(n, (hq + 2 * hkv) * d, dtype=dtype, device="cuda").normal_(0, 2, generator=gen)
    blocks = -(-n // BS) if case["append"] else 1
    pool_k = torch.empty(1, blocks + 1, hkv, BS, d, dtype=dtype, device="cuda").normal_(generator=gen)
    pool_v = torch.empty_like(pool_k).normal_(generator=gen)
    weight = [torch.empty(d, dtype=dtype, device="cuda").normal_(1, 0.2, generator=gen) if case["norm"] else None
              for _ in range(2)]
    positions = _gpu(rng.randint(0, case["far"], (case["axes"], n)), torch.int64)
    return dict(pool_k=pool_k, pool_v=pool_v, qkv=qkv, hq=hq, interleaved=case["interleaved"], q_weight=weight[0],
                k_weight=weight[1], positions=positions if case["axes"] > 1 else positions[0],
                axes=_gpu(_pair_axes(half, case["axes"]), torch.int32) if case["axes"] > 1 else None,
                freq=_gpu(1e6 ** (-np.arange(half) / half), torch.float64),
                slots=_gpu(rng.permutation(blocks * BS)[:n], torch.int64) if case["append"] else None)


def _prepare_experts(case, rng, gen):
    t, h, i, e = case["tokens"], case["hidden"], case["inter"], case["experts"]
    dtype = DTYPES[case["dtype"]]

    def normal(std, *shape):
        return torch.empty(*shape, dtype=dtype, device="cuda").normal_(0, std, generator=gen)

    return dict(x=normal(1.0, t, h), router=normal(h ** -0.5, e, h), gate_up=normal(h ** -0.5, e, 2 * i, h),
                down=normal(i ** -0.5, e, h, i), top=case["top"])


PREPARE = {"positions": _prepare_positions, "rotary": _prepare_rotary, "experts": _prepare_experts}


# ---------------------------------------------------------------- one pass

def run(s):
    if own:
        return OWN[s["op"]](s)
    return PLAIN[s["op"]](s)


def _own_positions(s):
    from mini_inference_b200 import ops
    return ops.media_positions(s["positions"], s["media"], s["media_counts"], s["seq_rows"], s["cu_seqlens"], out=s["out"])


def _own_rotary(s):
    from mini_inference_b200 import ops
    kw = dict(axes=s["axes"], q_weight=s["q_weight"], k_weight=s["k_weight"], eps=EPS, interleaved=s["interleaved"])
    if s["slots"] is not None:
        q, _, _ = ops.norm_rotary_append(s["pool"], 0, s["qkv"], s["positions"], s["freq"], s["hq"],
                                         slot_mapping=s["slots"], **kw)
        return q, s["pool_k"], s["pool_v"]
    return ops.norm_rotary_append(s["pool"], 0, s["qkv"], s["positions"], s["freq"], s["hq"], k_out=True, v_out=True, **kw)


def _own_experts(s):
    from mini_inference_b200 import ops
    return ops.expert_mlp(s["x"], s["router"], s["gate_up"], s["down"], s["top"], s["workspace"])


OWN = {"positions": _own_positions, "rotary": _own_rotary, "experts": _own_experts}


def _plain_positions(s):
    pos = s["positions"]
    token = torch.arange(pos.numel(), device="cuda")
    seq = torch.searchsorted(s["cu_seqlens"].long(), token, right=True) - 1
    row = s["seq_rows"].long()
    start, f, h, w, step = s["media"].long()[row].unbind(-1)  # [batch, spans] each
    there = torch.arange(start.shape[1], device="cuda") < s["media_counts"].long()[row][:, None]
    size = torch.where(there, f * h * w, 0)
    far = torch.where(there, torch.maximum(torch.maximum((f - 1) * step + 1, h), w), 0)
    before = (size - far).cumsum(1)  # by how much positions lag behind indexes after each span
    start = torch.where(there, start, 1 << 60)
    which = (start[seq] <= pos[:, None]).sum(1) - 1  # the last span that starts at or before the token
    j = which.clamp(min=0)
    at = [x[seq, j] for x in (start, size, far, before, h.clamp(min=1), w.clamp(min=1), step)]
    a, n, ahead, lag, hh, ww, st = at
    r = pos - a
    inside = (which >= 0) & (r < n)
    lag = torch.where(which >= 0, lag, 0)
    base = a - (lag - (n - ahead))
    frame, rest = torch.div(r, hh * ww, rounding_mode="floor"), r % (hh * ww)
    grid = (base + frame * st, base + torch.div(rest, ww, rounding_mode="floor"), base + rest % ww)
    return torch.stack([torch.where(inside, g, pos - lag) for g in grid])


def _plain_rotary(s):
    n = s["qkv"].shape[0]
    hkv, d = s["pool_k"].shape[2], s["pool_k"].shape[4]
    r = 2 * s["freq"].numel()
    pos = s["positions"].double()
    angle = (pos[:, None] if s["axes"] is None else pos[s["axes"].long()].T) * s["freq"]
    cos, sin = (f(angle).float()[:, None, :] for f in (torch.cos, torch.sin))
    x = s["qkv"].view(n, -1, d)
    heads = x[:, :s["hq"] + hkv].float()
    if s["q_weight"] is not None:
        unit = heads * torch.rsqrt((heads * heads).mean(-1, keepdim=True) + EPS)
        heads = torch.cat([unit[:, :s["hq"]] * s["q_weight"].float(), unit[:, s["hq"]:] * s["k_weight"].float()], 1)
    if s["interleaved"]:
        a, b = heads[..., 0:r:2], heads[..., 1:r:2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = heads[..., :r // 2], heads[..., r // 2:r]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    y = torch.cat([y, heads[..., r:]], -1).to(x.dtype)
    q, k, v = y[:, :s["hq"]], y[:, s["hq"]:], x[:, s["hq"] + hkv:]
    if s["slots"] is None:
        return q.contiguous(), k.contiguous(), v.contiguous()
    s["pool_k"][0, s["slots"] // BS, :, s["slots"] % BS] = k
    s["pool_v"][0, s["slots"] // BS, :, s["slots"] % BS] = v
    return q.contiguous(), s["pool_k"], s["pool_v"]


def _plain_experts(s):
    x = s["x"].float()
    t, inter = x.shape[0], s["down"].shape[2]
    # In 64 bits: a choice between two experts that are almost alike hangs on the last bits.
    logits = s["x"].double() @ s["router"].double().T
    expert = logits.sort(dim=-1, descending=True, stable=True).indices[:, :s["top"]]
    weight = torch.softmax(logits, -1).gather(1, expert)
    weight = (weight / weight.sum(-1, keepdim=True)).float()
    if expert.numel() < s["router"].shape[0]:  # few tokens: the chosen experts' weights for each
        pick = expert.flatten()
        h = (s["gate_up"][pick].float() @ x.repeat_interleave(s["top"], 0)[:, :, None])[..., 0]
        h = h[:, :inter] * torch.sigmoid(h[:, :inter]) * h[:, inter:]
        y = (s["down"][pick].float() @ h[:, :, None])[..., 0].view(t, s["top"], -1)
        return (y * weight[:, :, None]).sum(1).to(s["x"].dtype)
    h = x @ s["gate_up"].float().transpose(1, 2)  # every expert on every token
    h = h[..., :inter] * torch.sigmoid(h[..., :inter]) * h[..., inter:]
    share = torch.zeros(t, s["router"].shape[0], device="cuda").scatter(1, expert, weight)
    y = (h * share.T[:, :, None]) @ s["down"].float().transpose(1, 2)
    return y.sum(0).to(s["x"].dtype)


PLAIN = {"positions": _plain_positions, "rotary": _plain_rotary, "experts": _plain_experts}


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    if case["op"] == "positions":
        n = int(_spread(case["new_lo"], case["new_hi"], case["batch"]).sum())
        return {"bytes": n * 32 + case["batch"] * (12 + 20 * case["spans"]), "flops": n * 10}
    if case["op"] == "rotary":
        hq, hkv, d = SHAPES[case["shape"]]
        n = case["rows"]
        return {"bytes": n * (2 * (hq + 2 * hkv) * d * 2 + 8 * case["axes"] + (8 if case["append"] else 0)) + 8 * d,
                "flops": n * (hq + hkv) * (3 * case["rotary"] + 4 * d)}
    t, h, i, e, k = case["tokens"], case["hidden"], case["inter"], case["experts"], case["top"]
    touched = e * (1 - (1 - k / e) ** t)  # experts that at least one token chooses, of choices at random
    return {"bytes": int(touched * 3 * h * i * 2 + e * h * 2 + 2 * t * h * 2), "flops": t * (6 * k * h * i + 2 * e * h)}


# ---------------------------------------------------------------- from the definitions, in 64 bits

def exact(case, seed):
    if case["op"] == "rotary":
        return _exact_rotary(prepare(case, seed))
    if case["op"] == "experts":
        return _exact_experts(prepare(case, seed))
    return None  # whole numbers


def _exact_rotary(s):
    n, hkv, d = s["qkv"].shape[0], s["pool_k"].shape[2], s["pool_k"].shape[4]
    half = s["freq"].numel()
    at = s["positions"] if s["axes"] is None else s["positions"][s["axes"].long()]
    turn = at.double()[:, None] * s["freq"] if s["axes"] is None else at.double().T * s["freq"]
    z = torch.polar(torch.ones_like(turn), turn)[:, None, :]
    y = s["qkv"].double().view(n, -1, d).clone()
    if s["q_weight"] is not None:
        for heads, w in ((slice(0, s["hq"]), s["q_weight"]), (slice(s["hq"], s["hq"] + hkv), s["k_weight"])):
            size = torch.linalg.vector_norm(y[:, heads], dim=-1, keepdim=True)
            y[:, heads] = y[:, heads] / torch.sqrt(size ** 2 / d + EPS) * w.double()
    turned = slice(0, s["hq"] + hkv)
    x = y.clone()
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


def _exact_experts(s):
    x, inter = s["x"].double(), s["down"].shape[2]
    out = torch.zeros_like(x)
    logits = x @ s["router"].double().T
    chosen = torch.zeros_like(logits, dtype=torch.bool)
    left = logits.clone()
    for _ in range(s["top"]):  # the largest, the first among equals, one after another
        best = left == left.amax(1, keepdim=True)
        first = best & (best.cumsum(1) == 1)
        chosen |= first
        left[first] = -math.inf
    share = torch.softmax(logits.masked_fill(~chosen, -math.inf), -1)
    for e in range(s["router"].shape[0]):
        at = chosen[:, e].nonzero()[:, 0]
        if at.numel():
            h = x[at] @ s["gate_up"][e].double().T
            h = torch.nn.functional.silu(h[:, :inter]) * h[:, inter:]
            out[at] += share[at, e, None] * (h @ s["down"][e].double().T)
    return out
