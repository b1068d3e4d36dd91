"""ops.norm_rotary_append: head norms, rotation by one axis or several, and the append, in float64.

Tolerance of one element, u half a step of the storage type and f the attention factor. The norm:
the sum of d squares (all positive) is off by at most d 2^-24 of itself, its root by half of that;
rsqrtf by two units (2^-22), the two products by one half step each: (d / 2 + 8) 2^-24 of the
normalised element. The rotation adds, as in the rotation without norm, 2^-20 f (|a| + |b|) of the
pair. The output is rounded once: u of itself, and float16's smallest step 2^-25.
"""

from __future__ import annotations

import pytest
import torch

from mini_inference_b200 import PkvError, ops

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def reference(x, positions, freq, axes, weight, eps, interleaved, factor):
    """(values, bound before rounding) of heads x [N, H, d]."""
    d, half = x.shape[-1], freq.numel()
    y = x.double()
    norm = 0.0
    if weight is not None:
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()
        norm = (d / 2 + 8) * 2.0 ** -24
    pos = positions.double()
    angle = (pos[:, None] if axes is None else pos[axes.long()].T) * freq
    c, s = angle.cos()[:, None] * factor, angle.sin()[:, None] * factor
    first, second = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    a, b = y[..., first], y[..., second]
    out, bound = y.clone(), norm * y.abs()
    out[..., first], out[..., second] = a * c - b * s, b * c + a * s
    bound[..., first] = bound[..., second] = (2.0 ** -20 + norm) * factor * (a.abs() + b.abs())
    return out, bound


def check(got, x, *args):
    want, bound = reference(x, *args)
    u = torch.finfo(got.dtype).eps / 2
    excess = (got.double() - want).abs() - (u * (want.abs() + bound) + bound + 2.0 ** -25)
    assert (excess <= 0).all(), excess.max().item()


def setup(dtype, hq, hkv, d, n, axes, *, far=40000, extra=0, seed=0, blocks=9, bs=16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    width = (hq + 2 * hkv) * d
    qkv = (torch.randn(n, width + extra, generator=g, device="cuda") * 2).to(dtype)[:, :width]
    pos = torch.randint(0, far, (axes, n), generator=g, device="cuda")
    if n:
        pos[:, 0], pos[:, -1] = 0, far - 1
    weights = [torch.randn(d, generator=g, device="cuda").to(dtype) for _ in range(2)]
    k = torch.full((2, blocks + 1, hkv, bs, d), 5.0, dtype=dtype, device="cuda")
    return qkv, pos if axes > 1 else pos[0], weights, k, torch.full_like(k, 6.0)


@pytest.mark.parametrize("dtype,hq,hkv,d", [(F16, 14, 2, 64), (BF16, 28, 4, 128), (F16, 3, 1, 80), (BF16, 4, 4, 36),
                                            (BF16, 2, 1, 512), (F16, 8, 2, 256), (BF16, 6, 3, 72), (F16, 5, 5, 16)])
@pytest.mark.parametrize("part", [1.0, 0.5])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("axes,norm", [(1, True), (3, True), (2, False)])
@pytest.mark.parametrize("n,extra", [(1, 0), (67, 3), (130, 8)])
def test_layouts(dtype, hq, hkv, d, part, interleaved, axes, norm, n, extra):
    rotary = int(d * part) // 2 * 2
    qkv, pos, (qw, kw), k, v = setup(dtype, hq, hkv, d, n, axes, extra=extra, seed=n)
    if not norm:
        qw = kw = None
    half = rotary // 2
    freq, _ = ops.rotary_frequencies(rotary, 1e6)
    sections = [half] if axes == 1 else [half - (axes - 1) * (half // axes)] + [half // axes] * (axes - 1)
    pair = ops.pair_axes(sections, alternate=n > 1) if axes > 1 else None
    slots = torch.randperm(9 * 16, device="cuda")[:n]
    if n > 2:
        slots[1] = -1  # skipped
    q, ko, vo = ops.norm_rotary_append(ops.make_pool(k, v), 1, qkv, pos, freq, hq, axes=pair, q_weight=qw, k_weight=kw, eps=1e-5,
                                       interleaved=interleaved, attention_factor=1.25, k_out=True, v_out=True,
                                       slot_mapping=slots)
    heads = qkv.reshape(n, -1, d)
    check(q, heads[:, :hq], pos, freq, pair, qw, 1e-5, interleaved, 1.25)
    check(ko, heads[:, hq:hq + hkv], pos, freq, pair, kw, 1e-5, interleaved, 1.25)
    assert torch.equal(vo, heads[:, hq + hkv:])
    at = slots >= 0
    assert torch.equal(k[1, slots[at] // 16, :, slots[at] % 16], ko[at])
    assert torch.equal(v[1, slots[at] // 16, :, slots[at] % 16], vo[at])
    rest = torch.ones(10 * 16, dtype=torch.bool, device="cuda")
    rest[slots[at]] = False
    assert (k[0] == 5).all() and (v[0] == 6).all()
    flat = k[1].transpose(1, 2).reshape(-1, hkv, d), v[1].transpose(1, 2).reshape(-1, hkv, d)
    assert (flat[0][rest] == 5).all() and (flat[1][rest] == 6).all()


def test_many_rows():
    qkv, pos, (qw, kw), k, v = setup(BF16, 28, 4, 128, 2500, 3, far=1 << 20, blocks=160)
    freq, _ = ops.rotary_frequencies(128, 1e6)
    pair = ops.pair_axes([16, 24, 24])
    slots = torch.randperm(160 * 16, device="cuda")[:2500]
    q, _, _ = ops.norm_rotary_append(ops.make_pool(k, v), 0, qkv, pos, freq, 28, axes=pair, q_weight=qw, k_weight=kw,
                                     slot_mapping=slots)
    heads = qkv.view(2500, -1, 128)
    check(q, heads[:, :28], pos, freq, pair, qw, 1e-6, False, 1.0)
    check(k[0, slots // 16, :, slots % 16], heads[:, 28:32], pos, freq, pair, kw, 1e-6, False, 1.0)
    assert torch.equal(v[0, slots // 16, :, slots % 16], heads[:, 32:])


@pytest.mark.parametrize("interleaved", [False, True])
def test_without_norm_it_is_rotary_append(interleaved):
    qkv, pos, _, k, v = setup(F16, 14, 2, 64, 33, 1)
    pool = ops.make_pool(k, v)
    freq, _ = ops.rotary_frequencies(32, 1e4)
    want = ops.rotary_append(pool, 0, qkv, pos, freq, 14, interleaved=interleaved, k_out=True, v_out=True)
    got = ops.norm_rotary_append(pool, 0, qkv, pos, freq, 14, interleaved=interleaved, k_out=True, v_out=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # Axes that agree are one axis.
    pair = ops.pair_axes([4, 6, 6])
    got = ops.norm_rotary_append(pool, 0, qkv, pos.expand(3, -1).contiguous(), freq, 14, axes=pair, interleaved=interleaved,
                                 k_out=True, v_out=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("d", [64, 36])
def test_in_place(d):
    qkv, pos, (qw, kw), k, v = setup(BF16, 8, 2, d, 40, 1)
    pool = ops.make_pool(k, v)
    freq, _ = ops.rotary_frequencies(d, 1e4)
    q, ko, vo = ops.norm_rotary_append(pool, 0, qkv, pos, freq, 8, q_weight=qw, k_weight=kw, k_out=True, v_out=True)
    rows = qkv.clone()
    heads = rows.view(40, -1, d)
    ops.norm_rotary_append(pool, 0, rows, pos, freq, 8, q_weight=qw, k_weight=kw, q_out=heads[:, :8], k_out=heads[:, 8:10],
                           v_out=heads[:, 10:])
    assert torch.equal(heads[:, :8], q) and torch.equal(heads[:, 8:10], ko) and torch.equal(heads[:, 10:], vo)


def test_rows_of_zeros_and_of_large_values():
    """A head of zeros stays zero; squares past float16's range are float32's."""
    qkv, pos, (qw, kw), k, v = setup(F16, 4, 2, 64, 5, 1)
    qkv[1] = 0
    qkv[2] *= 10000
    freq, _ = ops.rotary_frequencies(64, 1e4)
    q, ko, _ = ops.norm_rotary_append(ops.make_pool(k, v), 0, qkv, pos, freq, 4, q_weight=qw, k_weight=kw, k_out=True)
    assert (q[1] == 0).all() and (ko[1] == 0).all()
    check(q, qkv.view(5, -1, 64)[:, :4], pos, freq, None, qw, 1e-6, False, 1.0)
    qkv[3, 7] = float("nan")  # of q head 0: the others do not see it
    again, _, _ = ops.norm_rotary_append(ops.make_pool(k, v), 0, qkv, pos, freq, 4, q_weight=qw, k_weight=kw, k_out=True)
    assert again[3, 0].isnan().all() and torch.equal(again[3, 1:], q[3, 1:]) and torch.equal(again[[0, 1, 2, 4]], q[[0, 1, 2, 4]])


def test_reports_and_refusals():
    qkv, pos, (qw, kw), k, v = setup(F16, 14, 2, 64, 8, 3)
    pool = ops.make_pool(k, v)
    freq, _ = ops.rotary_frequencies(64, 1e4)
    pair = ops.pair_axes([8, 12, 12])
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    ok = dict(pool=pool, layer=0, qkv=qkv, positions=pos, inv_freq=freq, num_q_heads=14, axes=pair, q_weight=qw, k_weight=kw,
              k_out=True, status=status)
    ops.norm_rotary_append(**ok)
    ops.raise_device_errors(status)
    slots = torch.arange(8, device="cuda")
    slots[3] = 10 * 16
    wrong = pair.clone()
    wrong[5] = 3
    for kw_ in (dict(slot_mapping=slots), dict(axes=wrong), dict(positions=pos - 1)):
        ops.norm_rotary_append(**{**ok, **kw_})
        with pytest.raises(IndexError):
            ops.raise_device_errors(status)
    for kw_ in (dict(qkv=qkv[:, :-1]), dict(qkv=qkv.bfloat16()), dict(positions=pos.int()), dict(positions=pos[:, :3].contiguous()),
                dict(inv_freq=freq.float()), dict(axes=None), dict(axes=pair[:5]), dict(axes=pair.long()), dict(q_weight=None),
                dict(k_weight=kw[:32]), dict(k_weight=kw.float()), dict(slot_mapping=slots[:4]),
                dict(positions=pos.view(3, 2, 4)), dict(q_out=torch.empty(8, 13, 64, device="cuda"))):
        with pytest.raises(ValueError):
            ops.norm_rotary_append(**{**ok, **kw_})
    for kw_ in (dict(k_out=False), dict(eps=-1.0), dict(eps=float("nan")), dict(layer=2, slot_mapping=slots),
                dict(positions=pos.repeat(2, 1))):
        with pytest.raises(PkvError):
            ops.norm_rotary_append(**{**ok, **kw_})
    assert ops.norm_rotary_append(**{**ok, "qkv": qkv[:0], "positions": pos[:, :0].contiguous()})[0].shape == (0, 14, 64)


@pytest.mark.parametrize("dtype,d,rotary", [(F16, 64, 32), (BF16, 128, 32), (F16, 80, 16), (BF16, 72, 16), (F16, 36, 18)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_infinity_and_nan_past_the_rotated_part(dtype, d, rotary, interleaved, norm, bad):
    """One bad element in the part that is not rotated, at each of its places: without norms every other element is as it was."""
    n = d - rotary
    qkv, pos, (qw, kw), k, v = setup(dtype, 4, 2, d, n, 3, seed=d)
    heads = qkv.view(n, -1, d)
    at = torch.arange(n, device="cuda")
    heads[at, 1, rotary + at] = bad  # q head 1
    heads[at, 4, rotary + at] = bad  # k head 0
    heads[at, 5, rotary + at] = -0.0
    freq, _ = ops.rotary_frequencies(rotary, 1e4)
    third = rotary // 6
    pair = ops.pair_axes([rotary // 2 - 2 * third, third, third])
    if not norm:
        qw = kw = None
    q, ko, _ = ops.norm_rotary_append(ops.make_pool(k, v), 0, qkv, pos, freq, 4, axes=pair, q_weight=qw, k_weight=kw,
                                      interleaved=interleaved, k_out=True)
    for got, x, w in ((q, heads[:, :4], qw), (ko, heads[:, 4:6], kw)):
        want, bound = reference(x, pos, freq, pair, w, 1e-6, interleaved, 1.0)
        assert torch.equal(got.isnan(), want.isnan())
        if not norm:
            assert torch.equal(got[..., rotary:].nan_to_num(7, 8, 9).view(torch.int16),
                               x[..., rotary:].nan_to_num(7, 8, 9).view(torch.int16))
        fine = want.isfinite()
        off = (got.double() - want).abs()[fine]
        u = torch.finfo(dtype).eps / 2
        assert (off <= (u * (want.abs() + bound) + bound + 2.0 ** -25)[fine]).all()
        assert (got.isinf() == want.isinf()).all()
