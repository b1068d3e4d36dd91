"""ops.expert_mlp (router and experts of a decoder layer) against its definition in float64."""

from __future__ import annotations

import pytest
import torch

from mini_inference_b200 import PkvError, ops

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16]


def make(dtype, tokens, hidden, inter, experts, seed=0, dev="cuda"):
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(std, *shape):
        return torch.empty(*shape, dtype=dtype, device=dev).normal_(0, std, generator=g)

    return (normal(1.0, tokens, hidden), normal(hidden ** -0.5, experts, hidden),
            normal(hidden ** -0.5, experts, 2 * inter, hidden), normal(inter ** -0.5, experts, hidden, inter))


def choose(logits, top_k):
    """The experts of the largest logits, the first among equals."""
    return logits.sort(dim=-1, descending=True, stable=True).indices[:, :top_k]


def reference(x, router, gate_up, down, top_k, renormalize=True):
    """(out, bound) in float64: the result and what the roundings may add to it.

    With u half a step of the type, relative: silu(gate) * up is rounded once (u of each activation)
    and so is the result; float32 sums of n products are off by at most n 2^-24 of the sum of the
    products' sizes (twice that here: the tensor core's adds may cut instead of rounding), gate's
    error passes silu with a slope below 1.1, and __expf adds 2^-20 of silu.
    """
    u = torch.finfo(x.dtype).eps / 2
    xd = x.double()
    logits = xd @ router.double().T
    chosen = choose(logits, top_k)
    share = torch.softmax(logits, -1).gather(1, chosen)
    if renormalize:
        share = share / share.sum(-1, keepdim=True)
    inter, hidden = down.shape[2], down.shape[1]
    out, bound = torch.zeros_like(xd), torch.zeros_like(xd)
    eps1, eps2 = hidden * 2.0 ** -23, inter * 2.0 ** -23
    for e in range(router.shape[0]):
        at, k = (chosen == e).nonzero(as_tuple=True)
        if not at.numel():
            continue
        w = gate_up[e].double()
        h, size = xd[at] @ w.T, xd[at].abs() @ w.abs().T
        gate, up = h[:, :inter], h[:, inter:]
        act = torch.nn.functional.silu(gate) * up
        off = (1.1 * size[:, :inter] * up.abs() + torch.nn.functional.silu(gate).abs() * size[:, inter:]) * eps1
        off = off + act.abs() * (u + 2.0 ** -20) + torch.finfo(x.dtype).tiny * u
        d = down[e].double()
        y, ysize = act @ d.T, act.abs() @ d.abs().T
        s = share[at, k, None]
        out.index_add_(0, at, s * y)
        bound.index_add_(0, at, s * (off @ d.abs().T + ysize * (eps2 + 2.0 ** -20)))
    return out, bound * 1.01 + out.abs() * u * 1.01 + torch.finfo(x.dtype).tiny * u


def check(x, router, gate_up, down, top_k, renormalize=True, workspace=None, **kw):
    t, h = x.shape[0], x.shape[1]
    ws = workspace if workspace is not None else ops.expert_mlp_workspace(t, router.shape[0], top_k, h, down.shape[2], x.device)
    status = torch.zeros(1, dtype=torch.int32, device=x.device)
    got = ops.expert_mlp(x, router, gate_up, down, top_k, ws, renormalize=renormalize, status=status, **kw)
    ops.raise_device_errors(status)
    want, bound = reference(x, router, gate_up, down, top_k, renormalize)
    excess = ((got.double() - want).abs() - bound).max().item()
    assert excess <= 0, excess
    assert not ws[:6200].any()  # ready for the next call
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,hidden,inter,experts,top_k", [
    (1, 64, 64, 4, 2), (1, 896, 608, 8, 2), (1, 2048, 768, 64, 8), (2, 128, 8, 1, 1), (3, 8, 40, 5, 5), (7, 896, 1216, 32, 4),
    (16, 1000, 1000, 16, 2), (17, 200, 136, 512, 16), (64, 2048, 1024, 64, 8), (65, 512, 96, 100, 3), (255, 264, 72, 6, 2),
])
def test_few_tokens(dtype, tokens, hidden, inter, experts, top_k):
    check(*make(dtype, tokens, hidden, inter, experts), top_k)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,hidden,inter,experts,top_k", [
    (20, 8, 16, 5, 2), (9, 64, 8, 3, 1), (128, 512, 104, 7, 3), (129, 512, 112, 7, 3), (200, 40, 24, 2, 2), (300, 8, 8, 9, 9),
    (256, 512, 256, 4, 1), (257, 512, 264, 4, 4), (333, 896, 616, 60, 4), (1025, 256, 200, 3, 2), (2048, 1024, 384, 128, 8),
])
def test_many_tokens(dtype, tokens, hidden, inter, experts, top_k):
    check(*make(dtype, tokens, hidden, inter, experts), top_k)


@pytest.mark.parametrize("renormalize", [True, False])
def test_weights_of_the_chosen_or_of_all(renormalize):
    x, router, gate_up, down = make(torch.float16, 33, 256, 128, 16)
    check(x, router * 4, gate_up, down, 3, renormalize)


@pytest.mark.parametrize("tokens,hidden,top_k", [(1031, 576, 8), (1031, 1040, 8), (911, 544, 9), (700, 1024, 16)])
def test_large_products_one_call_after_another(tokens, hidden, top_k):
    """16 MB of products and more, whose lines are dropped where they are whole (hidden a multiple of 32)."""
    ws = ops.expert_mlp_workspace(tokens, 24, top_k, hidden, 64, "cuda")
    for seed in range(3):
        check(*make(torch.bfloat16, tokens - 40 * seed, hidden, 64, 24, seed=seed), top_k, workspace=ws)


@pytest.mark.parametrize("tokens", [96, 97, 113, 128, 129, 193, 224, 225, 241, 256, 257, 385, 512, 513])
def test_tiles_at_the_edges_of_their_copies(tokens):
    """One expert, so that the tiles' sizes are known: rows come 128 or 32 at a time."""
    check(*make(torch.float16, tokens, 136, 72, 1, seed=tokens), 1)


def test_all_tokens_to_one_expert():
    """An expert with every token (several tiles of them) and experts with none."""
    x, router, gate_up, down = make(torch.bfloat16, 700, 256, 128, 8)
    x[:, 0] = 8
    router.zero_()
    router[5, 0] = 1
    check(x, router, gate_up, down, 1)


@pytest.mark.parametrize("tokens", [5, 40, 150])
def test_equal_logits_go_to_the_first(tokens):
    """Twin experts and tokens of zeros: the lowest indexes are taken."""
    x, router, gate_up, down = make(torch.float16, tokens, 128, 64, 12)
    x[::3] = 0
    router[7] = router[2]
    router[11] = router[2]
    check(x, router, gate_up, down, 4)


def test_near_ties_are_decided_by_exact_logits():
    """Experts whose logits differ by less than float32 sums tell apart."""
    g = torch.Generator(device="cuda").manual_seed(3)
    hidden, experts = 2048, 32
    x, _, gate_up, down = make(torch.float16, 64, hidden, 64, experts, seed=1)
    base = torch.empty(hidden, device="cuda").normal_(0, 0.02, generator=g).half()
    router = base.repeat(experts, 1)
    # One small element of each row moved by its last bit: logits about 2^-22 of their size apart.
    at = base.abs().argsort()[:experts]
    router[torch.arange(experts, device="cuda"), at] = base[at] + base[at].abs() * 2.0 ** -10
    logits = x.double() @ router.double().T
    order = logits.sort(-1, descending=True).values
    assert ((order[:, 3] - order[:, 4]) < 1e-5).any()
    check(x, router, gate_up, down, 4)


@pytest.mark.parametrize("tokens", [8, 40, 150])
def test_one_tokens_nan_and_infinity_stay_its_own(tokens):
    x, router, gate_up, down = make(torch.float16, tokens, 256, 128, 8)
    clean = check(x, router, gate_up, down, 2)
    bad = x.clone()
    bad[3, 5] = float("nan")
    bad[6, 7] = float("inf")
    ws = ops.expert_mlp_workspace(tokens, 8, 2, 256, 128, "cuda")
    got = ops.expert_mlp(bad, router, gate_up, down, 2, ws)
    keep = [i for i in range(tokens) if i not in (3, 6)]
    assert torch.equal(got[keep], clean[keep])
    assert got[3].isnan().all()


def test_strides_shapes_and_given_output():
    x, router, gate_up, down = make(torch.bfloat16, 24, 128, 64, 4)
    wide = torch.full((24, 200), float("nan"), dtype=x.dtype, device="cuda")
    wide[:, :128] = x
    want = check(x, router, gate_up, down, 2)
    ws = ops.expert_mlp_workspace(24, 4, 2, 128, 64, "cuda")
    assert torch.equal(ops.expert_mlp(wide[:, :128], router, gate_up, down, 2, ws), want)
    odd = torch.empty(24 * 128 + 1, dtype=x.dtype, device="cuda")[1:].view(24, 128).copy_(x)  # not on 16 bytes
    assert torch.equal(ops.expert_mlp(odd, router, gate_up, down, 2, ws), want)
    assert torch.equal(ops.expert_mlp(x.T.contiguous().T, router, gate_up, down, 2, ws), want)
    out = torch.empty(2, 12, 128, dtype=x.dtype, device="cuda")
    assert ops.expert_mlp(x.view(2, 12, 128), router, gate_up, down, 2, ws, out=out) is not None
    assert torch.equal(out.view(24, 128), want)
    assert ops.expert_mlp(x[:0], router, gate_up, down, 2, ws).shape == (0, 128)


def test_a_workspace_serves_calls_of_every_size():
    """Larger and smaller calls and other shapes through one workspace, each as alone; twice the same bits."""
    big = make(torch.float16, 600, 256, 264, 16)
    small = make(torch.float16, 3, 896, 128, 64, seed=5)
    ws = torch.zeros(max(ops.expert_mlp_workspace(600, 16, 4, 256, 264, "cuda").numel(),
                         ops.expert_mlp_workspace(3, 64, 8, 896, 128, "cuda").numel()), dtype=torch.uint8, device="cuda")
    first = check(*big, 4, workspace=ws)
    check(*small, 8, workspace=ws)
    assert torch.equal(check(*big, 4, workspace=ws), first)
    ws[6400:] = 255  # what is behind the counters may hold anything
    assert torch.equal(check(*big, 4, workspace=ws), first)


def test_values_past_float16_overflow_as_they_are_rounded():
    """Activations past the type's range are infinite, as silu(gate) * up is when it is rounded; nothing else is."""
    x, router, gate_up, down = make(torch.float16, 6, 64, 32, 4)
    gate_up[:, 0] = 60  # gate row 0 and up row 0 of every expert: about 60 |x| each, their product far past 65504
    gate_up[:, 32] = 60
    x = x.abs() * 4
    for t in (1, 6):
        ws = ops.expert_mlp_workspace(t, 4, 2, 64, 32, "cuda")
        got = ops.expert_mlp(x[:t], router, gate_up, down, 2, ws)
        assert not got.isfinite().any()
    down[:, :, 0] = 0  # infinity times nothing
    assert ops.expert_mlp(x, router, gate_up, down, 2, ws).isnan().all()


@pytest.mark.parametrize("tokens", [6, 32, 200])
def test_captured_and_replayed_on_other_inputs(tokens):
    x, router, gate_up, down = make(torch.bfloat16, tokens, 512, 256, 16)
    ws = ops.expert_mlp_workspace(tokens, 16, 4, 512, 256, "cuda")
    out = torch.empty_like(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.expert_mlp(x, router, gate_up, down, 4, ws, out=out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.expert_mlp(x, router, gate_up, down, 4, ws, out=out)
        ops.expert_mlp(out, router, gate_up, down, 4, ws)
    for seed in (1, 2, 3):
        x.copy_(make(torch.bfloat16, tokens, 512, 256, 16, seed=seed)[0])
        graph.replay()
        assert torch.equal(out, check(x, router, gate_up, down, 4))


def test_two_calls_at_once_on_two_streams():
    """Each with its own workspace: CTAs of both share the GPU."""
    a, b = make(torch.float16, 64, 512, 512, 32), make(torch.float16, 5, 1024, 256, 16, seed=2)
    want_a, want_b = check(*a, 4), check(*b, 2)
    ws_a = ops.expert_mlp_workspace(64, 32, 4, 512, 512, "cuda")
    ws_b = ops.expert_mlp_workspace(5, 16, 2, 1024, 256, "cuda")
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(50):
        with torch.cuda.stream(streams[0]):
            got[0].append(ops.expert_mlp(*a, 4, ws_a))
        with torch.cuda.stream(streams[1]):
            got[1].append(ops.expert_mlp(*b, 2, ws_b))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want_a) for g in got[0]) and all(torch.equal(g, want_b) for g in got[1])


def test_refusals():
    x, router, gate_up, down = make(torch.float16, 12, 128, 64, 4)
    ws = ops.expert_mlp_workspace(12, 4, 2, 128, 64, "cuda")
    ok = dict(x=x, router=router, gate_up=gate_up, down=down, top_k=2, workspace=ws)
    for kw in (dict(router=router[:, :64].contiguous()), dict(router=router.float()), dict(gate_up=gate_up[:, :64].contiguous()),
               dict(down=down[:2].contiguous()), dict(down=down.transpose(1, 2)), dict(x=x.bfloat16()), dict(workspace=ws.cpu()),
               dict(out=torch.empty(12, 64, dtype=x.dtype, device="cuda")), dict(out=torch.empty(128, 12, dtype=x.dtype, device="cuda").T),
               dict(workspace=ws.view(-1, 2)[:, 0]), dict(router=router.cpu())):
        with pytest.raises(ValueError):
            ops.expert_mlp(**{**ok, **kw})
    with pytest.raises(NotImplementedError):
        ops.expert_mlp(**{**ok, "x": x.float()})
    for kw in (dict(top_k=5), dict(top_k=0), dict(workspace=ws[:-256])):
        with pytest.raises(PkvError):
            ops.expert_mlp(**{**ok, **kw})
    odd = make(torch.float16, 4, 100, 64, 4)
    with pytest.raises(PkvError):
        ops.expert_mlp(*odd, 2, ws)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,hidden,inter,experts,top_k", [
    (1, 2048, 768, 64, 8), (8, 896, 608, 8, 2), (16, 1000, 1000, 16, 2), (64, 512, 1024, 16, 4), (100, 512, 136, 3, 2), (128, 512, 520, 2, 1),
    (200, 640, 416, 3, 2), (333, 896, 616, 60, 4), (1025, 256, 200, 3, 2), (700, 512, 1024, 2, 1), (2048, 1024, 384, 16, 4),
])
def test_nothing_but_the_result_is_rounded(dtype, tokens, hidden, inter, experts, top_k):
    """The error, as a 2-norm, is that of rounding the exact result to the type.

    What the two halves of an activation leave (2^-17 of it in bfloat16, 2^-22 in float16), the float32 sums
    (2^-20 of the result) and the weights are a tenth of that rounding (some 2^-9.5 and 2^-12.5) at most, and a
    tenth beside one in a 2-norm adds a tenth. An activation rounded once would bring it to 1.4, and so would one
    more rounding of gate and up.
    """
    x, router, gate_up, down = make(dtype, tokens, hidden, inter, experts, seed=tokens)
    ws = ops.expert_mlp_workspace(tokens, experts, top_k, hidden, inter, "cuda")
    got = ops.expert_mlp(x, router, gate_up, down, top_k, ws).double()
    want, _ = reference(x, router, gate_up, down, top_k)
    off, rounding = (got - want).norm(), (want.to(dtype).double() - want).norm()
    assert off <= 1.1 * rounding, (off / rounding).item()


@pytest.mark.parametrize("tokens,hidden,inter,experts,top_k", [(333, 896, 616, 60, 4), (1500, 256, 1024, 24, 4), (400, 512, 512, 8, 2), (2048, 512, 768, 64, 8)])
def test_the_same_bits_every_time_whatever_the_experts_loads(tokens, hidden, inter, experts, top_k):
    """Experts of every load, some with several tiles of which the last is smaller: rows go to them in no fixed order."""
    x, router, gate_up, down = make(torch.bfloat16, tokens, hidden, inter, experts, seed=3)
    x[:, 0] = 1
    router[:, 0] = torch.linspace(-1.5, 1.5, experts, device="cuda")
    first = check(x, router, gate_up, down, top_k)
    for t in (tokens - 7, tokens):  # other calls of the same size, other loads
        want = check(x[:t], router, gate_up, down, top_k)
        for _ in range(12):
            ws = ops.expert_mlp_workspace(t, experts, top_k, hidden, inter, "cuda")
            assert torch.equal(ops.expert_mlp(x[:t], router, gate_up, down, top_k, ws), want)
    assert torch.equal(first, want)
