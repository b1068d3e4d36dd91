"""pkv_tree_attention: drafted trees over the paged cache, against the definition in float64.

Tolerance of one output element, from the roundings the kernel makes (u = half a step of the
storage type, A = sum_j p_j |v_j| / sum_j p_j over the visible keys, n of them):

* the weights are rounded to the storage type: u A (and, for float16, half of its smallest
  step, 2^-25, per key where a weight is subnormal; the sum of weights is at least 1/2);
* the output is rounded once: u |out|;
* a score is a float32 sum of d products and two more roundings: off by at most
  delta = (d + 4) 2^-24 scale sum |q_i k_i| + 2^-21 (the exponential's own error), so
  weights and their sum are off by delta each: 2 delta A, with the largest delta of the row;
* the products with V and the sum of weights add n + 1 terms in float32, each rounded or
  cut to 2^-23: 2 n 2^-23 A.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

BS = 16


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA GPU")
    return torch.device("cuda", 0)


def pack_mask(vis: list[torch.Tensor], words: int) -> torch.Tensor:
    """Boolean [T, T] per tree -> int64 [N, words]."""
    rows = []
    for v in vis:
        t = v.shape[0]
        bits = torch.zeros(t, words * 64, dtype=torch.int64)
        bits[:, :t] = v.long()
        rows.append((bits.view(t, words, 64) << torch.arange(64)).sum(-1))
    return torch.cat(rows) if rows else torch.zeros(0, words, dtype=torch.int64)


def tree_visible(t: int, branch: int) -> torch.Tensor:
    vis = torch.eye(t, dtype=torch.bool)
    for i in range(1, t):
        vis[i] |= vis[(i - 1) // branch]
    return vis


class Case:
    def __init__(self, dev, dtype, hq, hkv, d, ctx, nodes, *, branch=2, vis=None, layers=1, layer=0, seed=0, spread=1.0,
                 extra_blocks=3, poison=True):
        g = torch.Generator().manual_seed(seed)
        self.dtype, self.hq, self.hkv, self.d, self.layer = dtype, hq, hkv, d, layer
        need = [-(-c // BS) for c in ctx]
        total = sum(need) + extra_blocks
        order = torch.randperm(total, generator=g)
        cols = max(1, max(need, default=1))
        tables = torch.full((max(1, len(ctx)), cols), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            tables[b, :n] = order[at:at + n].int()
            at += n
        shape = (layers, total + 1, hkv, BS, d)
        self.k = (torch.randn(shape, generator=g) * spread).to(dtype).to(dev)
        self.v = torch.randn(shape, generator=g).to(dtype).to(dev)
        if poison:  # what no sequence holds may be anything
            for b, c in enumerate(ctx):
                if c % BS:
                    self.k[:, tables[b, c // BS], :, c % BS:] = float("nan")
                    self.v[:, tables[b, c // BS], :, c % BS:] = float("inf")
            self.k[:, total] = float("nan")
            self.v[:, total] = float("nan")
        self.ctx, self.nodes = ctx, nodes
        n = sum(nodes)
        self.q = (torch.randn(n, hq, d, generator=g) * spread).to(dtype).to(dev)
        self.kn = (torch.randn(n, hkv, d, generator=g) * spread).to(dtype).to(dev)
        self.vn = torch.randn(n, hkv, d, generator=g).to(dtype).to(dev)
        self.vis = vis if vis is not None else [tree_visible(t, branch) for t in nodes]
        self.words = max(1, -(-max(nodes, default=1) // 64))
        self.mask = pack_mask(self.vis, self.words).to(dev)
        self.tables = tables.to(dev)
        self.cu = torch.tensor([0] + list(torch.tensor(nodes).cumsum(0)) if nodes else [0], dtype=torch.int32, device=dev)
        self.lens = torch.tensor(ctx, dtype=torch.int32, device=dev)
        self.dev = dev

    def run(self, *, seq_rows=None, scale=None, workspace=None, max_nodes=None, **kw):
        from mini_inference_b200 import ops

        pool = ops.make_pool(self.k, self.v)
        ws = workspace if workspace is not None else ops.tree_attention_workspace(pool, max(1, len(self.ctx)), self.dev)
        status = torch.zeros(1, dtype=torch.int32, device=self.dev)
        args = {"q": self.q, "k_nodes": self.kn, "v_nodes": self.vn, **kw}
        out = ops.tree_attention(pool, self.layer, ops.make_tables(self.tables, seq_rows), args["q"], args["k_nodes"],
                                 args["v_nodes"], self.cu, self.lens, self.mask,
                                 max(self.nodes, default=0) if max_nodes is None else max_nodes, ws,
                                 out=args.get("out"), scale=scale, status=status)
        ops.raise_device_errors(status)
        return out

    def expected(self, scale=None):
        """(out, tolerance) in float64."""
        scale = self.d ** -0.5 if scale is None else scale
        u = torch.finfo(self.dtype).eps / 2
        tiny = 2.0 ** -25 if self.dtype == torch.float16 else 0.0
        out = torch.zeros(self.q.shape, dtype=torch.float64, device=self.dev)
        tol = torch.zeros_like(out)
        lo = 0
        for b, t in enumerate(self.nodes):
            c = self.ctx[b]
            blocks = self.tables[b, :-(-c // BS)].long()
            for h in range(self.hkv):
                k = torch.cat([self.k[self.layer, blocks, h].reshape(-1, self.d)[:c], self.kn[lo:lo + t, h]]).double()
                v = torch.cat([self.v[self.layer, blocks, h].reshape(-1, self.d)[:c], self.vn[lo:lo + t, h]]).double()
                vis = torch.cat([torch.ones(t, c, dtype=torch.bool), self.vis[b]], 1).to(self.dev)
                group = self.hq // self.hkv
                for gq in range(h * group, (h + 1) * group):
                    q = self.q[lo:lo + t, gq].double()
                    s = (q @ k.T * scale).masked_fill(~vis, float("-inf"))
                    p = torch.nan_to_num(torch.softmax(s, -1), nan=0.0)
                    a = p @ v.abs()
                    size = ((q.abs() @ k.abs().T) * scale).masked_fill(~vis, 0.0).amax(-1, keepdim=True)
                    delta = (self.d + 4) * 2.0 ** -24 * size + 2.0 ** -21
                    n = vis.sum(-1, keepdim=True).double()
                    o = p @ v
                    out[lo:lo + t, gq] = o
                    tol[lo:lo + t, gq] = (u * o.abs() + (u + 2 * delta + 2 * n * 2.0 ** -23) * a
                                          + 2 * tiny * (vis.double() @ v.abs()) + 2.0 ** -25)
            lo += t
        return out, tol

    def check(self, out, scale=None, rows=slice(None)):
        want, tol = self.expected(scale)
        off = ((out.double() - want).abs() - tol)[rows]
        assert torch.isfinite(out[rows]).all()
        assert off.max().item() <= 0, f"{off.max().item():.3e} past the tolerance at {off.argmax().item()}"


SHAPES = [(torch.float16, 14, 2, 64), (torch.bfloat16, 28, 4, 128), (torch.bfloat16, 14, 2, 64),
          (torch.float16, 28, 4, 128)]


@pytest.mark.parametrize("dtype,hq,hkv,d", SHAPES)
@pytest.mark.parametrize("ctx,nodes", [
    ([33], [5]), ([0], [1]), ([0], [7]), ([1], [1]), ([15, 16, 17], [3, 1, 2]), ([63, 64, 65, 0], [18, 19, 36, 37]),
    ([130, 700, 5], [8, 0, 64]), ([1000], [65]), ([257, 40], [128, 129]), ([2500], [16]), ([6001, 31], [9, 33])])
def test_matches_the_definition(dev, dtype, hq, hkv, d, ctx, nodes):
    case = Case(dev, dtype, hq, hkv, d, ctx, nodes, seed=len(ctx) + sum(nodes))
    case.check(case.run())


@pytest.mark.parametrize("hq,hkv,d", [(1, 1, 64), (2, 2, 64), (6, 2, 128), (16, 2, 64), (16, 1, 128), (18, 2, 64),
                                      (32, 8, 128), (33, 3, 64), (80, 5, 128)])
def test_head_layouts(dev, hq, hkv, d):
    case = Case(dev, torch.bfloat16, hq, hkv, d, [77, 400], [21, 6], branch=3, seed=hq)
    case.check(case.run())


@pytest.mark.parametrize("dtype,hq,hkv,d", SHAPES[:2])
def test_widest_trees_and_chains(dev, dtype, hq, hkv, d):
    case = Case(dev, dtype, hq, hkv, d, [300, 65, 0], [512, 100, 512], branch=1, seed=3)
    case.check(case.run())


@pytest.mark.parametrize("dtype,hq,hkv,d", SHAPES[:2])
@pytest.mark.parametrize("batch,ctx", [(1, 20000), (3, 9000), (40, 333), (200, 40)])
def test_every_way_of_splitting(dev, dtype, hq, hkv, d, batch, ctx):
    lens = [max(0, ctx - 37 * b) for b in range(batch)]
    case = Case(dev, dtype, hq, hkv, d, lens, [1 + b % 11 for b in range(batch)], seed=batch)
    case.check(case.run())


@pytest.mark.parametrize("dtype,hq,hkv,d", SHAPES[:2])
def test_any_mask_and_rows_that_see_nothing(dev, dtype, hq, hkv, d):
    g = torch.Generator().manual_seed(9)
    nodes, ctx = [70, 5, 130], [0, 0, 50]
    vis = [torch.rand(t, t, generator=g) < 0.3 for t in nodes]
    vis[0][3] = False
    vis[0][69] = False
    vis[1][:] = False
    vis[2][7] = False  # sees its context alone
    case = Case(dev, dtype, hq, hkv, d, ctx, nodes, vis=vis, seed=4)
    out = case.run()
    case.check(out)
    assert (out[3] == 0).all() and (out[69] == 0).all() and (out[70:75] == 0).all()


@pytest.mark.parametrize("dtype,hq,hkv,d", SHAPES[:2])
def test_nodes_that_no_one_sees_may_hold_anything(dev, dtype, hq, hkv, d):
    """Trees padded to one size: the padding's K/V are whatever the buffers held."""
    nodes, real = [12, 150, 64, 90], [5, 130, 1, 0]
    vis = []
    for t, n in zip(nodes, real):
        see = torch.zeros(t, t, dtype=torch.bool)
        see[:n, :n] = tree_visible(n, 2)[:n, :n] if n else False
        vis.append(see)
    case = Case(dev, dtype, hq, hkv, d, [40, 333, 0, 16], nodes, vis=vis)
    lo = 0
    clean_k, clean_v = case.kn.clone(), case.vn.clone()
    for t, n in zip(nodes, real):
        case.kn[lo + n:lo + t] = float("nan")
        case.vn[lo + n:lo + t, :, ::2] = float("inf")
        case.vn[lo + n:lo + t, :, 1::2] = float("nan")
        lo += t
    out = case.run()
    case.kn, case.vn = clean_k, clean_v  # unseen: the values make no difference
    case.check(out)


@pytest.mark.parametrize("dtype,hq,hkv,d", SHAPES[:2])
def test_large_scores_move_the_maximum(dev, dtype, hq, hkv, d):
    case = Case(dev, dtype, hq, hkv, d, [900, 64], [20, 3], spread=4.0, seed=5)
    case.check(case.run())
    case = Case(dev, dtype, hq, hkv, d, [900, 4096], [20, 3], seed=6)
    case.check(case.run(scale=0.5), scale=0.5)


@pytest.mark.parametrize("dtype,hq,hkv,d", SHAPES[:2])
def test_strides_and_views(dev, dtype, hq, hkv, d):
    case = Case(dev, dtype, hq, hkv, d, [100, 31], [9, 20], seed=7)
    want = case.run()
    n = sum(case.nodes)
    # The projection's rows: q and v as their columns, k a permuted copy.
    rows = torch.zeros(n, (hq + 2 * hkv) * d, dtype=dtype, device=dev)
    rows[:, :hq * d] = case.q.flatten(1)
    rows[:, (hq + hkv) * d:] = case.vn.flatten(1)
    k = case.kn.transpose(0, 1).contiguous().transpose(0, 1)
    got = case.run(q=rows[:, :hq * d].view(n, hq, d), k_nodes=k, v_nodes=rows[:, (hq + hkv) * d:].view(n, hkv, d))
    assert torch.equal(got, want)
    # One node's rows, and one head's, for all (stride 0): copied by the wrapper.
    same = Case(dev, dtype, hq, hkv, d, [100, 31], [9, 20], seed=7)
    same.kn, same.vn = case.kn[:1].expand(n, hkv, d), case.vn[:, :1].expand(n, hkv, d)
    same.check(same.run())
    # Rows on 4 bytes only: q and out by pairs, k and v copied by the wrapper.
    def odd(x):
        base = torch.zeros(n, x.shape[1] * d + 2, dtype=dtype, device=dev)
        base[:, 2:] = x.flatten(1)
        return base[:, 2:].view(n, x.shape[1], d)

    buf = torch.full((n + 2, hq * d + 2), 7.0, dtype=dtype, device=dev)
    out = buf[1:-1, 2:].view(n, hq, d)
    got = case.run(q=odd(case.q), k_nodes=odd(case.kn), v_nodes=odd(case.vn), out=out)
    assert torch.equal(got, want) and got.data_ptr() == out.data_ptr()
    assert (buf[0] == 7).all() and (buf[-1] == 7).all() and (buf[:, :2] == 7).all()


def test_padding_rows_layers_and_rows_behind(dev):
    """Table rows by slot, a padding sequence, another layer, and nodes behind the last tree."""
    case = Case(dev, torch.float16, 14, 2, 64, [50, 90, 20], [4, 6, 3], layers=3, layer=2, seed=8)
    base = case.run()
    case.check(base)
    perm = torch.tensor([2, 0, 1], device=dev)
    slots = torch.full((5, case.tables.shape[1]), -1, dtype=torch.int32, device=dev)
    slots[perm + 1] = case.tables
    plain, case.tables = case.tables, slots
    rows = (perm + 1).int()
    assert torch.equal(case.run(seq_rows=rows), base)
    # The second sequence turned into padding: its nodes see their tree alone.
    rows[1] = -1
    got = case.run(seq_rows=rows)
    case.tables = plain
    case.check(got, rows=[*range(4), *range(10, 13)])  # (where keys are split depends on the whole batch)
    alone = Case(dev, torch.float16, 14, 2, 64, [0], [6], seed=8)
    alone.q, alone.kn, alone.vn = case.q[4:10].contiguous(), case.kn[4:10].contiguous(), case.vn[4:10].contiguous()
    alone.check(got[4:10])
    # Fewer trees than node rows: what lies behind the last one stays.
    case2 = Case(dev, torch.float16, 14, 2, 64, [50, 90, 20], [4, 6, 3], layers=3, layer=2, seed=8)
    case2.cu = torch.tensor([0, 4, 10, 10], dtype=torch.int32, device=dev)
    out = torch.full_like(case2.q, 3.0)
    case2.run(out=out)
    case.check(out, rows=slice(0, 10))
    assert (out[10:] == 3).all()


def test_the_same_result_each_time_and_from_a_graph(dev):
    from mini_inference_b200 import ops

    case = Case(dev, torch.bfloat16, 28, 4, 128, [3000, 700, 64], [12, 3, 40], seed=10)
    pool = ops.make_pool(case.k, case.v)
    ws = ops.tree_attention_workspace(pool, 3, dev)
    want = case.run(workspace=ws)
    for _ in range(3):
        assert torch.equal(case.run(workspace=ws), want)
    tables = ops.make_tables(case.tables)
    outs = [torch.zeros_like(want) for _ in range(2)]
    graphs = []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for out in outs:  # two graphs over one workspace, replayed in turn
        with torch.cuda.stream(side):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                ops.tree_attention(pool, 0, tables, case.q, case.kn, case.vn, case.cu, case.lens, case.mask, 40, ws, out=out)
            graphs.append(g)
    torch.cuda.synchronize()
    for g in graphs:
        g.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want) and torch.equal(outs[1], want)
    # Other lengths on the device, the same graphs: the split follows them.
    case.lens.copy_(torch.tensor([5, 700, 33], dtype=torch.int32))
    graphs[0].replay()
    torch.cuda.synchronize()
    case.ctx = [5, 700, 33]
    case.check(outs[0])


def test_two_calls_at_once(dev):
    """Calls on two streams, a workspace each, with other work on the GPU between them."""
    from mini_inference_b200 import ops

    cases = [Case(dev, torch.bfloat16, 28, 4, 128, [3000, 5000, 100, 7000], [16, 40, 16, 7], seed=1),
             Case(dev, torch.float16, 14, 2, 64, [300] * 40, [9] * 40, seed=2)]
    spaces = [ops.tree_attention_workspace(ops.make_pool(c.k, c.v), 64, dev) for c in cases]
    want = [c.run() for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(30):
        for i, c in enumerate(cases):
            status = torch.zeros(1, dtype=torch.int32, device=dev)
            streams[i].wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(streams[i]):
                out = ops.tree_attention(ops.make_pool(c.k, c.v), 0, ops.make_tables(c.tables), c.q, c.kn, c.vn, c.cu, c.lens,
                                         c.mask, max(c.nodes), spaces[i], status=status)
            outs[i].append((out, status))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(s.item() == 0 and torch.equal(o, want[i]) for o, s in outs[i])


def test_cache_past_32_bit_offsets(dev):
    hkv, d, blocks = 8, 128, 131080  # 2^31 elements and a little more
    k = torch.zeros(1, blocks + 1, hkv, BS, d, dtype=torch.bfloat16, device=dev)
    v = torch.zeros_like(k)
    case = Case(dev, torch.bfloat16, 32, hkv, d, [70], [5], seed=11)
    base = case.run()
    used = case.tables[0].long()
    high = torch.arange(blocks - used.numel(), blocks, device=dev)
    k[0, high], v[0, high] = case.k[0, used], case.v[0, used]
    case.k, case.v, case.tables = k, v, high.int()[None].contiguous()
    assert torch.equal(case.run(), base)


def test_bad_indexes_are_reported(dev):
    def bad(**kw):
        case = Case(dev, torch.float16, 14, 2, 64, [50, 20], [4, 6], seed=12)
        for name, value in kw.items():
            setattr(case, name, torch.tensor(value, dtype=torch.int32, device=dev))
        with pytest.raises(IndexError):
            case.run()

    bad(lens=[50, 20000])
    bad(lens=[-1, 20])
    bad(cu=[0, 4, 11])
    bad(cu=[4, 0, 10])
    bad(tables=[[0, 1, 2, 99], [3, 4, 0, 0]])
    bad(tables=[[0, -1, 2, 3], [3, 4, 0, 0]])
    case = Case(dev, torch.float16, 14, 2, 64, [50, 20], [4, 6], seed=12)
    for most in (5, 0):
        with pytest.raises(IndexError):
            case.run(max_nodes=most)
    with pytest.raises(IndexError):
        case.run(seq_rows=torch.tensor([0, 2], dtype=torch.int32, device=dev))


def test_refusals(dev):
    from mini_inference_b200 import PkvError, ops

    case = Case(dev, torch.float16, 14, 2, 64, [50], [4], seed=13)
    pool, tables = ops.make_pool(case.k, case.v), ops.make_tables(case.tables)
    ws = ops.tree_attention_workspace(pool, 1, dev)

    def call(**kw):
        a = dict(q=case.q, kn=case.kn, vn=case.vn, cu=case.cu, lens=case.lens, mask=case.mask, most=4, ws=ws, scale=None) | kw
        return ops.tree_attention(pool, 0, tables, a["q"], a["kn"], a["vn"], a["cu"], a["lens"], a["mask"], a["most"], a["ws"],
                                  scale=a["scale"])

    for kw in (dict(q=case.q.bfloat16()), dict(kn=case.kn[:3]), dict(cu=case.cu.long()), dict(mask=case.mask.int()),
               dict(mask=case.mask[:3]), dict(lens=case.lens.float())):
        with pytest.raises(ValueError):
            call(**kw)
    for kw in (dict(most=65), dict(scale=0.0), dict(scale=float("nan")), dict(ws=ws[256:]), dict(ws=ws[8:])):
        with pytest.raises(PkvError):
            call(**kw)
    with pytest.raises(RuntimeError):
        call(q=case.q.cpu())
    with pytest.raises(ValueError):
        ops.tree_attention_workspace(pool, 1025, dev)
    assert call(q=case.q[:0], kn=case.kn[:0], vn=case.vn[:0], mask=case.mask[:0], cu=case.cu * 0).shape == (0, 14, 64)
