"""Which experts ops.expert_mlp chooses, seen in its outputs: the largest logits by float64, the first among equals."""

from __future__ import annotations

import pytest
import torch

from mini_inference_b200 import ops

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16]


def signed_experts(dtype, experts, hidden):
    """gate_up and down of experts whose output is their weight times silu(8) at their own place, for tokens with x[0] = 1."""
    gate_up = torch.zeros(experts, 16, hidden, dtype=dtype, device="cuda")
    gate_up[:, 0, 0], gate_up[:, 8, 0] = 8, 1
    down = torch.zeros(experts, hidden, 8, dtype=dtype, device="cuda")
    down[torch.arange(experts), torch.arange(experts), 0] = 1
    return gate_up, down


def check_choice(x, router, top_k, batch):
    """Calls of ``batch`` tokens each; every token's set of experts is that of its float64 logits."""
    experts, hidden = router.shape
    gate_up, down = signed_experts(x.dtype, experts, hidden)
    ws = ops.expert_mlp_workspace(batch, experts, top_k, hidden, 8, "cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = torch.cat([ops.expert_mlp(x[a:a + batch], router, gate_up, down, top_k, ws, status=status)
                     for a in range(0, x.shape[0], batch)])
    ops.raise_device_errors(status)
    logits = x.double() @ router.double().T
    want = torch.zeros_like(logits, dtype=torch.bool)
    want.scatter_(1, logits.sort(dim=-1, descending=True, stable=True).indices[:, :top_k], True)
    wrong = ((got[:, :experts] != 0) != want).any(-1).nonzero()[:, 0]
    assert not wrong.numel(), (wrong[:8].tolist(), logits[wrong[:4]].tolist())
    assert not got[:, experts:].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch", [7, 40, 150])  # one launch; tokens loaded whole; laid out by expert
@pytest.mark.parametrize("twins", [1, 2])
def test_logits_at_every_step_from_the_border(dtype, batch, twins):
    """Logits 1 + j 2^-23 beside the last chosen one's 1, for every j up to past where the border may end.

    All are exact in float32 in any order of their sum. One expert so placed, or two; the largest logit, from
    which the border's width may come, in several sizes.
    """
    hidden, top_k = 64, 2 + twins
    tops = (1.25, 1.2578125, 1.26171875, 1.33203125)
    steps = 256
    router = torch.zeros(3 + twins, hidden, dtype=dtype, device="cuda")
    router[0, 1:5] = torch.tensor([1.0, 1 / 4, 1 / 128, 1 / 256])  # with x[2:5] what the largest logit is made of
    router[1:, 5] = 1
    router[1:1 + twins, 6] = 2.0 ** -23
    x = torch.zeros(len(tops) * steps, hidden, dtype=dtype, device="cuda")
    x[:, 0] = x[:, 1] = x[:, 5] = 1
    x[:, 6] = torch.arange(steps, device="cuda").repeat(len(tops))
    for i, top in enumerate(tops):
        part = x[i * steps:(i + 1) * steps]
        n = round((top - 1.25) * 256)
        part[:, 2], part[:, 3], part[:, 4] = 1, n // 2, n % 2
    assert (x.double() @ router.double().T)[:, 0].unique().tolist() == sorted(tops)
    check_choice(x, router, top_k, batch)
    check_choice(x.flip(0), router, top_k, batch)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,hidden", [(5, 2048), (40, 2048), (150, 2048), (7, 1000), (130, 1000)])
@pytest.mark.parametrize("infinite", [False, True])
def test_near_ties_behind_large_terms_that_cancel(dtype, batch, hidden, infinite):
    """Pairs of opposite channels of some thousand, which float32 sums do not come back from to a logit's last bits.

    Experts' rows differ by the last bits of a few elements, so that logits of size 1 are some 2^-13 apart; partial
    sums past 2048 are rounded to 2^-12 or 2^-13. One more expert whose logit is minus infinity changes nothing.
    """
    g = torch.Generator(device="cuda").manual_seed(11)
    experts, top_k, tokens = 32, 4, 300
    u = torch.finfo(dtype).eps
    base = (torch.randn(hidden, generator=g, device="cuda") * hidden ** -0.5).to(dtype)
    few = 64 if dtype == torch.float16 else 8
    moved = (torch.rand(experts, hidden, generator=g, device="cuda") < few / hidden) & (base.abs() > 2.0 ** -12)
    sign = torch.randint(0, 2, (experts, hidden), generator=g, device="cuda") * 2 - 1
    router = (base.float() * (1 + moved * sign * u)).to(dtype)
    x = torch.randn(tokens, hidden, generator=g, device="cuda").to(dtype)
    pairs = 10 + torch.randperm(hidden - 10, generator=g, device="cuda")[:8].view(2, 4)
    large = (4096 * (1 + torch.rand(tokens, 4, generator=g, device="cuda"))).to(dtype)
    x[:, pairs[0]], x[:, pairs[1]] = large, -large
    common = torch.rand(experts, 4, generator=g, device="cuda").add(0.5).to(dtype)
    router[:, pairs[0]] = router[:, pairs[1]] = common
    x[:, 0], router[:, 0] = 1, 0
    if infinite:
        router[5, 1], x[:, 1] = -torch.inf, 1
    check_choice(x[:tokens // batch * batch], router, top_k, batch)
