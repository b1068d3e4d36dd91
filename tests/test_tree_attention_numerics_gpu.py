"""pkv_tree_attention's softmax weights: the bits they keep, small ones beside a large one, every key once.

The tolerances count the roundings of tests/test_tree_attention_gpu.py (u = half a step of the
storage type, A = sum_j p_j |v_j|, n visible keys, delta the error of a score), but with the weights as
they are meant to reach the products with V:

* bfloat16: two halves, the first cut (off by less than 2 u), the second that remainder rounded (off by
  u of it), so a weight is off by 2 u u of itself;
* float16: one half, off by u of itself down to 2^-25 of the row's running maximum. (The weights
  are made 2^11 times as large, so the smallest normal number, 2^-14, stands for 2^-25.)
"""

from __future__ import annotations

import pytest
import torch

from tests.test_tree_attention_gpu import BS, Case, SHAPES

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA GPU")
    return torch.device("cuda", 0)


def expected(case, weight, scale=None):
    """(out, tolerance) in float64 where a weight is off by `weight` of itself."""
    u = torch.finfo(case.dtype).eps / 2
    scale = case.d ** -0.5 if scale is None else scale
    out = torch.zeros(case.q.shape, dtype=torch.float64, device=case.dev)
    tol = torch.zeros_like(out)
    group, lo = case.hq // case.hkv, 0
    for b, t in enumerate(case.nodes):
        c = case.ctx[b]
        blocks = case.tables[b, :-(-c // BS)].long()
        vis = torch.cat([torch.ones(t, c, dtype=torch.bool), case.vis[b]], 1).to(case.dev)
        for h in range(case.hq):
            kv = h // group
            k = torch.cat([case.k[case.layer, blocks, kv].reshape(-1, case.d)[:c], case.kn[lo:lo + t, kv]]).double()
            v = torch.cat([case.v[case.layer, blocks, kv].reshape(-1, case.d)[:c], case.vn[lo:lo + t, kv]]).double()
            q = case.q[lo:lo + t, h].double()
            p = torch.softmax((q @ k.T * scale).masked_fill(~vis, float("-inf")), -1)
            size = ((q.abs() @ k.abs().T) * scale).masked_fill(~vis, 0.0).amax(-1, keepdim=True)
            delta = (case.d + 4) * 2.0 ** -24 * size + 2.0 ** -21
            n = vis.sum(-1, keepdim=True).double()
            out[lo:lo + t, h] = o = p @ v
            tol[lo:lo + t, h] = u * o.abs() + (weight + 2 * delta + 2 * n * 2.0 ** -23) * (p @ v.abs()) + 2.0 ** -25
        lo += t
    return out, tol


@pytest.mark.parametrize("hq,hkv,d", [(28, 4, 128), (14, 2, 64)])
@pytest.mark.parametrize("ctx,nodes", [([3, 40, 0], [1, 9, 12]), ([200], [100])])
def test_bfloat16_weights_keep_two_halves(dev, hq, hkv, d, ctx, nodes):
    case = Case(dev, torch.bfloat16, hq, hkv, d, ctx, nodes, seed=31)
    want, tol = expected(case, 2 * (torch.finfo(torch.bfloat16).eps / 2) ** 2)
    off = (case.run().double() - want).abs() - tol
    assert off.max().item() <= 0, off.max().item()


@pytest.mark.parametrize("dtype,hq,hkv,d", SHAPES)
@pytest.mark.parametrize("below", [12.5, 15.0, 16.5, 17.25])
def test_a_long_tail_beside_dominant_keys_of_no_value(dev, dtype, hq, hkv, d, below):
    """The first key of every other block scores `below` (18 to 24.9 in log2) above all others and has value zero: the others make the output.

    Scores are exact: q is one number in the first column, the keys' first column 0 or -below.
    """
    case = Case(dev, dtype, hq, hkv, d, [2000], [3], seed=32, poison=False)
    case.q.zero_()
    case.q[..., 0] = 8.0  # times the scale of 1/8: one
    case.k[..., 1:], case.kn[..., 1:] = 0.0, 0.0
    case.k[..., 0], case.kn[..., 0] = -below, -below
    case.k[:, 1::2, :, 0, 0] = 0.0  # the first key of every other block, blocks in any order
    case.v.abs_().mul_(4096.0)  # so that what is left of them is no subnormal output
    case.vn.abs_().mul_(4096.0)
    dominant = case.k[..., 0] == 0
    assert int(dominant.sum()) // hkv > 50
    case.v[dominant] = 0.0
    u = torch.finfo(dtype).eps / 2
    want, tol = expected(case, u if dtype == torch.float16 else 2 * u * u, scale=0.125)
    assert (tol < 0.01 * want).all()
    off = (case.run(scale=0.125).double() - want).abs() - tol
    assert off.max().item() <= 0, f"{(off / want).max().item():.3e} of the value past the tolerance"


@pytest.mark.parametrize("dtype,hq,hkv,d", SHAPES[:2])
@pytest.mark.parametrize("ctx,nodes", [([20000], [5]), ([20000], [64]), ([9000, 8999, 8961], [3, 1, 7]), ([500] * 60, [2] * 60)])
def test_every_stage_of_keys_counts_once(dev, dtype, hq, hkv, d, ctx, nodes):
    """Equal scores, and a value of one at the keys of one stage of 64 alone, another stage for each column and head.

    The sums are whole numbers, exact in float32; the exponentials and the quotient are
    within 2^-20 of it, and it is stored with one rounding.
    """
    case = Case(dev, dtype, hq, hkv, d, ctx, nodes, seed=33, poison=False)
    case.q.zero_()
    case.v.zero_()
    case.vn.zero_()
    per = hkv * d
    for b, c in enumerate(ctx):
        at = torch.arange(c, device=dev)
        blocks = case.tables[b].long()[at // BS]
        mark = at // 64 % per
        case.v[0, blocks, mark // d, at % BS, mark % d] = 1.0
    out = case.run().double()
    u, lo = torch.finfo(dtype).eps / 2, 0
    for b, (c, t) in enumerate(zip(ctx, nodes)):
        count = torch.zeros(per, dtype=torch.float64, device=dev)
        count.index_add_(0, torch.arange(c, device=dev) // 64 % per, torch.ones(c, dtype=torch.float64, device=dev))
        seen = c + case.vis[b].sum(-1).double().to(dev)
        want = count.view(1, hkv, 1, d) / seen.view(t, 1, 1, 1)
        got = out[lo:lo + t].view(t, hkv, hq // hkv, d)
        assert ((got - want).abs() <= (u + 2.0 ** -20) * want + 2.0 ** -25).all()
        lo += t


def test_nothing_is_computed_from_node_offsets_out_of_order(dev):
    """Trees that would overlap are reported and no output is written: their stages are not bounded by the nodes."""
    case = Case(dev, torch.float16, 14, 2, 64, [50, 20, 9], [4, 6, 2], seed=34)
    for cu in ([0, 10, 4, 12], [4, 0, 10, 12], [0, 4, 12, 10]):
        case.cu = torch.tensor(cu, dtype=torch.int32, device=dev)
        out = torch.full_like(case.q, 3.0)
        with pytest.raises(IndexError):
            case.run(out=out, max_nodes=12)
        assert (out == 3).all()
