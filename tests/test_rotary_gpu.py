"""pkv_rotary_append: interleaved and half layouts, part of the head, scaled frequencies; in float64.

Tolerance of one rotated element x c - y s with |(x, y)| the pair's length and f the attention
factor: the output is rounded once (u |out|, u half a step of the storage type); cos and sin are
off by the fraction of a turn rounded to float32 (half of 2^-24 turns, pi 2^-24) and two units of
2^-24 for the function and the factor; two products and a sum add three more roundings:
(4 + pi + 3) 2^-24 f (|x| + |y|), taken as 2^-20 f (|x| + |y|); float16's smallest step adds 2^-25.
"""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA GPU")
    return torch.device("cuda", 0)


def rotated(x, positions, freq, interleaved, factor):
    """(values, sizes) of the heads x [N, H, d] in float64."""
    x, half = x.double(), freq.numel()
    angle = (positions.double()[:, None] * freq)[:, None, :]
    c, s = angle.cos() * factor, angle.sin() * factor
    a, b = (x[..., 0:2 * half:2], x[..., 1:2 * half:2]) if interleaved else (x[..., :half], x[..., half:2 * half])
    out, size = x.clone(), torch.zeros_like(x)
    first, second = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    out[..., first], out[..., second] = a * c - b * s, b * c + a * s
    size[..., first] = size[..., second] = (a.abs() + b.abs()) * factor
    return out, size


def check(got, x, positions, freq, interleaved, factor):
    want, size = rotated(x, positions, freq, interleaved, factor)
    u = torch.finfo(got.dtype).eps / 2
    tol = u * want.abs() + 2.0 ** -20 * size + (size > 0) * 2.0 ** -25
    assert ((got.double() - want).abs() <= tol).all(), ((got.double() - want).abs() - tol).max().item()
    rest = 2 * freq.numel()
    assert torch.equal(got[..., rest:], x[..., rest:])


def setup(dev, dtype, hq, hkv, d, n, *, far=40000, extra=0, seed=0, layers=2, blocks=9, bs=16):
    g = torch.Generator(device=dev).manual_seed(seed)
    width = (hq + 2 * hkv) * d
    qkv = (torch.randn(n, width + extra, generator=g, device=dev) * 2).to(dtype)[:, :width]
    pos = torch.randint(0, far, (n,), generator=g, device=dev)
    if n:
        pos[0] = 0
        pos[-1] = far - 1
    k = torch.full((layers, blocks + 1, hkv, bs, d), 5.0, dtype=dtype, device=dev)
    return qkv, pos, k, torch.full_like(k, 6.0)


@pytest.mark.parametrize("dtype,hq,hkv,d", [(torch.float16, 14, 2, 64), (torch.bfloat16, 28, 4, 128),
                                            (torch.float16, 3, 1, 80), (torch.bfloat16, 4, 4, 36)])
@pytest.mark.parametrize("part", [1.0, 0.5, 0.25])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("n,extra", [(1, 0), (67, 0), (130, 3)])
def test_layouts(dev, dtype, hq, hkv, d, part, interleaved, n, extra):
    from mini_inference_b200 import ops

    rotary = int(d * part) // 2 * 2
    qkv, pos, k, v = setup(dev, dtype, hq, hkv, d, n, extra=extra, seed=n)
    freq, _ = ops.rotary_frequencies(rotary, 1e6, device=dev)
    pool = ops.make_pool(k, v)
    slots = torch.randperm(9 * 16, device=dev)[:n]
    if n > 2:
        slots[1] = -1  # skipped
    q, ko, vo = ops.rotary_append(pool, 1, qkv, pos, freq, hq, interleaved=interleaved, k_out=True, v_out=True,
                                  slot_mapping=slots)
    heads = qkv.reshape(n, -1, d)
    check(q, heads[:, :hq], pos, freq, interleaved, 1.0)
    check(ko, heads[:, hq:hq + hkv], pos, freq, interleaved, 1.0)
    assert torch.equal(vo, heads[:, hq + hkv:])
    at = slots >= 0
    assert torch.equal(k[1, slots[at] // 16, :, slots[at] % 16], ko[at])
    assert torch.equal(v[1, slots[at] // 16, :, slots[at] % 16], vo[at])
    rest = torch.ones(10 * 16, dtype=torch.bool, device=dev)
    rest[slots[at]] = False
    assert (k[0] == 5).all() and (v[0] == 6).all()
    flat = k[1].transpose(1, 2).reshape(-1, hkv, d), v[1].transpose(1, 2).reshape(-1, hkv, d)
    assert (flat[0][rest] == 5).all() and (flat[1][rest] == 6).all()


@pytest.mark.parametrize("far", [1 << 20, 1 << 30])
def test_far_positions_and_factor(dev, far):
    from mini_inference_b200 import ops

    qkv, pos, k, v = setup(dev, torch.bfloat16, 8, 2, 128, 50, far=far, seed=2)
    freq, factor = ops.rotary_frequencies(128, 1e6, ops.RopeScaling("yarn", 8.0), device=dev)
    assert factor == pytest.approx(0.1 * math.log(8.0) + 1)
    q, ko, _ = ops.rotary_append(ops.make_pool(k, v), 0, qkv, pos, freq, 8, attention_factor=factor, k_out=True)
    heads = qkv.view(50, -1, 128)
    check(q, heads[:, :8], pos, freq, False, factor)
    check(ko, heads[:, 8:10], pos, freq, False, factor)


@pytest.mark.parametrize("dtype,hq,hkv,d", [(torch.float16, 14, 2, 64), (torch.bfloat16, 28, 4, 128)])
def test_agrees_with_rope_append(dev, dtype, hq, hkv, d):
    """Whole heads in halves at unscaled frequencies: rope_append's result, whose tables and steps are rounded more."""
    from mini_inference_b200 import ops

    qkv, pos, k, v = setup(dev, dtype, hq, hkv, d, 64, far=4096, seed=3)
    pool = ops.make_pool(k, v)
    cos, sin = ops.rope_tables(d, 4096, 1e6, dtype, dev)
    want, _ = ops.rope_append(pool, 0, qkv, pos, cos, sin, hq, k_out=True)
    got, _, _ = ops.rotary_append(pool, 0, qkv, pos, ops.rotary_frequencies(d, 1e6, device=dev)[0], hq, k_out=True)
    _, size = rotated(qkv.view(64, -1, d)[:, :hq], pos, ops.rotary_frequencies(d, 1e6, device=dev)[0], False, 1.0)
    u = torch.finfo(dtype).eps / 2
    # rope_append: tables rounded (u each), products (u each), sum (u); its float32 frequencies and angles 4 half steps at 4096.
    assert ((got.double() - want.double()).abs() <= (5 * u + 4 * 4096 * 2.0 ** -24) * size + 2.0 ** -24).all()


@pytest.mark.parametrize("interleaved", [False, True])
def test_in_place_and_inverse(dev, interleaved):
    """Into the projection's own columns, and back by the frequencies' opposite."""
    from mini_inference_b200 import ops

    qkv, pos, k, v = setup(dev, torch.float16, 14, 2, 64, 33, seed=4)
    freq, _ = ops.rotary_frequencies(32, 1e4, device=dev)
    pool = ops.make_pool(k, v)
    q, ko, _ = ops.rotary_append(pool, 0, qkv, pos, freq, 14, interleaved=interleaved, k_out=True)
    rows = qkv.clone()
    heads = rows.view(33, -1, 64)
    ops.rotary_append(pool, 0, rows, pos, freq, 14, interleaved=interleaved, q_out=heads[:, :14], k_out=heads[:, 14:16])
    assert torch.equal(heads[:, :14], q) and torch.equal(heads[:, 14:16], ko)
    ops.rotary_append(pool, 0, rows, pos, -freq, 14, interleaved=interleaved, q_out=heads[:, :14], k_out=heads[:, 14:16])
    _, size = rotated(qkv.view(33, -1, 64), pos, freq, interleaved, 1.0)
    # two roundings of values of at most the pair's length
    assert ((rows.double() - qkv.double()).abs().view(33, -1, 64) <= 3 * 2.0 ** -11 * size + 2.0 ** -24).all()


def test_frequencies():
    from mini_inference_b200 import ops

    plain, one = ops.rotary_frequencies(64, 1e4, device="cpu")
    assert one == 1.0 and plain[0] == 1.0 and plain.dtype == torch.float64
    assert torch.allclose(plain, torch.tensor([1e4 ** (-2 * i / 64) for i in range(32)], dtype=torch.float64), rtol=1e-14)
    linear, _ = ops.rotary_frequencies(64, 1e4, ops.RopeScaling("linear", 4.0), device="cpu")
    assert torch.equal(linear, plain / 4)
    ntk, _ = ops.rotary_frequencies(64, 1e4, ops.RopeScaling("ntk", 4.0), device="cpu")
    assert ntk[0] == 1.0 and ntk[-1].item() == pytest.approx(plain[-1].item() / 4)
    yarn, factor = ops.rotary_frequencies(64, 1e4, ops.RopeScaling("yarn", 4.0, 4096), device="cpu")
    turns = plain * 4096 / (2 * math.pi)
    assert torch.allclose(yarn[turns > 64], plain[turns > 64]) and torch.allclose(yarn[turns < 0.5], plain[turns < 0.5] / 4)
    assert (yarn <= plain).all() and (yarn >= plain / 4 * (1 - 1e-12)).all() and factor == pytest.approx(1.1386294361)
    for bad in (dict(kind="other", factor=2.0), dict(kind="yarn", factor=0.5), dict(kind="yarn", factor=2.0, beta_fast=1.0)):
        with pytest.raises(ValueError):
            ops.RopeScaling(**bad)


def test_reports_and_refusals(dev):
    from mini_inference_b200 import PkvError, ops

    qkv, pos, k, v = setup(dev, torch.float16, 14, 2, 64, 8, seed=5)
    pool = ops.make_pool(k, v)
    freq, _ = ops.rotary_frequencies(64, 1e4, device=dev)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    slots = torch.arange(8, device=dev)
    slots[3] = 10 * 16
    ops.rotary_append(pool, 0, qkv, pos, freq, 14, slot_mapping=slots, status=status)
    with pytest.raises(IndexError):
        ops.raise_device_errors(status)
    for kw in (dict(qkv=qkv[:, :-1]), dict(qkv=qkv.bfloat16()), dict(positions=pos.int()), dict(positions=pos[:3]),
               dict(inv_freq=freq.float()), dict(slot_mapping=slots[:4]), dict(q_out=torch.empty(8, 13, 64, device=dev))):
        with pytest.raises(ValueError):
            ops.rotary_append(**{**dict(pool=pool, layer=0, qkv=qkv, positions=pos, inv_freq=freq, num_q_heads=14, k_out=True), **kw})
    for kw in (dict(k_out=False), dict(inv_freq=ops.rotary_frequencies(66, 1e4, device=dev)[0]),
               dict(slot_mapping=torch.arange(8, device=dev), layer=2)):
        with pytest.raises(PkvError):
            ops.rotary_append(**{**dict(pool=pool, layer=0, qkv=qkv, positions=pos, inv_freq=freq, num_q_heads=14, k_out=True), **kw})
    assert ops.rotary_append(pool, 0, qkv[:0], pos[:0], freq, 14, k_out=True)[0].shape == (0, 14, 64)
