"""Host-side refusals of the norm-rotation, media position and expert entry points: before any CUDA call, no GPU needed."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from mini_inference_b200 import _lib, ops

L = _lib.lib
OK, BAD, UNSUPPORTED, WORKSPACE = _lib.PKV_OK, _lib.PKV_ERR_INVALID_ARGUMENT, _lib.PKV_ERR_UNSUPPORTED, _lib.PKV_ERR_WORKSPACE
FAKE = 1 << 20  # aligned and never dereferenced: every call below is refused, or empty, on the host


def pool(**kw):
    a = dict(k=FAKE, v=FAKE, layers=2, blocks=9, hkv=2, bs=16, d=64, dtype=_lib.PKV_F16) | kw
    return ctypes.byref(_lib.PkvPool(*a.values()))


def test_norm_rotary_append():
    def call(p=None, layer=0, qkv=FAKE, stride=18 * 64, n=4, hq=14, pos=FAKE, pos_stride=4, axes=FAKE, num_axes=3, rotary=64,
             inter=0, qw=FAKE, kw=FAKE, eps=1e-6, q=FAKE, k=FAKE, slots=None):
        return L.pkv_norm_rotary_append(p or pool(), layer, qkv, stride, n, hq, pos, pos_stride, axes, num_axes, FAKE, rotary, inter,
                                        1.0, qw, kw, eps, q, 896, 64, k, 128, 64, None, 0, 0, slots, None, None)

    assert call(qkv=None) == BAD and call(q=None) == BAD and call(k=None) == BAD and call(n=-1) == BAD and call(hq=13) == BAD
    assert call(rotary=66) == BAD and call(rotary=0) == BAD and call(rotary=3) == BAD and call(inter=2) == BAD
    assert call(stride=17 * 64) == BAD and call(qkv=FAKE + 1) == BAD and call(pos=FAKE + 4) == BAD and call(axes=FAKE + 2) == BAD
    assert call(num_axes=0) == BAD and call(num_axes=5) == BAD and call(pos_stride=3) == BAD and call(axes=None) == BAD
    assert call(qw=None) == BAD and call(kw=None) == BAD and call(eps=-1.0) == BAD and call(eps=math.nan) == BAD
    assert call(layer=2, slots=FAKE) == BAD and call(pool(k=None), slots=FAKE) == BAD
    assert call(pool(dtype=7)) == UNSUPPORTED and call(pool(d=1024), stride=18 * 1024, rotary=1024) == UNSUPPORTED
    assert call(hq=1 << 24, stride=1 << 40) == UNSUPPORTED
    assert call(n=0, qkv=None) == OK


def test_media_positions():
    def call(pos=FAKE, n=4, cu=FAKE, seqs=2, media=FAKE, counts=FAKE, rows=3, spans=2, out=FAKE, stride=4):
        return L.pkv_media_positions(pos, n, cu, seqs, FAKE, media, counts, rows, spans, out, stride, None, None)

    assert call(pos=None) == BAD and call(out=None) == BAD and call(media=None) == BAD and call(counts=None) == BAD
    assert call(n=-1) == BAD and call(n=1 << 31) == BAD and call(seqs=-1) == BAD and call(rows=-1) == BAD and call(spans=-1) == BAD
    assert call(stride=3) == BAD and call(cu=None) == BAD and call(pos=FAKE + 4) == BAD and call(media=FAKE + 2) == BAD
    assert call(n=0) == OK


def test_expert_mlp():
    need = L.pkv_expert_mlp_workspace_bytes(16, 8, 2, 128, 64)
    assert need > 0 and need % 256 == 0
    for bad in ((16, 0, 1, 128, 64), (16, 513, 2, 128, 64), (16, 8, 9, 128, 64), (16, 32, 17, 128, 64), (16, 8, 0, 128, 64),
                (16, 8, 2, 129, 64), (16, 8, 2, 128, 60), (-1, 8, 2, 128, 64), (16, 8, 2, 0, 64)):
        assert L.pkv_expert_mlp_workspace_bytes(*bad) == 0
    grow = [L.pkv_expert_mlp_workspace_bytes(t, 8, 2, 128, 64) for t in (0, 1, 7, 16, 17, 64, 255, 256, 257, 300, 1000, 5000)]
    assert grow == sorted(grow)  # what holds a call holds every smaller one

    def call(dtype=_lib.PKV_BF16, x=FAKE, xs=128, n=16, hidden=128, inter=64, experts=8, top_k=2, router=FAKE, gu=FAKE, down=FAKE,
             out=FAKE, os=128, ws=FAKE, nbytes=need):
        return L.pkv_expert_mlp(dtype, x, xs, n, hidden, inter, experts, top_k, 1, router, gu, down, out, os, ws, nbytes, None, None)

    assert call(x=None) == BAD and call(router=None) == BAD and call(gu=None) == BAD and call(down=None) == BAD
    assert call(out=None) == BAD and call(ws=None) == BAD and call(n=-1) == BAD and call(top_k=9) == BAD and call(top_k=0) == BAD
    assert call(xs=120) == BAD and call(xs=130) == BAD and call(os=127) == BAD and call(x=FAKE + 8) == BAD
    assert call(gu=FAKE + 2) == BAD and call(ws=FAKE + 128) == BAD and call(hidden=0) == BAD and call(experts=-1) == BAD
    assert call(n=1 << 24, hidden=1 << 20, xs=1 << 20, os=1 << 20, inter=1 << 20, nbytes=1 << 62) == UNSUPPORTED
    assert L.pkv_expert_mlp_workspace_bytes(1 << 24, 8, 2, 1 << 20, 1 << 20) == 0
    assert call(dtype=5) == UNSUPPORTED and call(hidden=124) == UNSUPPORTED and call(inter=60) == UNSUPPORTED
    assert call(experts=600) == UNSUPPORTED and call(experts=64, top_k=17) == UNSUPPORTED
    assert call(nbytes=need - 1) == WORKSPACE and call(n=0, x=None, out=None) == OK


def test_pair_axes():
    assert ops.pair_axes([1, 2, 3], device="cpu").tolist() == [0, 1, 1, 2, 2, 2]
    assert ops.pair_axes([4, 2, 2], alternate=True, device="cpu").tolist() == [0, 1, 2, 0, 1, 2, 0, 0]
    assert ops.pair_axes([1, 2, 2], alternate=True, device="cpu").tolist() == [0, 1, 2, 1, 2]
    for bad in ([], [0, 0], [1, -1], [1] * 5):
        with pytest.raises(ValueError):
            ops.pair_axes(bad, device="cpu")


def test_wrappers_need_cuda_tensors():
    x, i = torch.zeros(1, 192, dtype=torch.float16), torch.zeros(1, dtype=torch.int32)
    p = _lib.PkvPool(FAKE, FAKE, 1, 1, 1, 16, 64, 0)
    with pytest.raises(RuntimeError):
        ops.norm_rotary_append(p, 0, x, i.long(), i.double(), 1)
    with pytest.raises(RuntimeError):
        ops.media_positions(i.long(), torch.zeros(1, 1, 5, dtype=torch.int32), i)
    with pytest.raises(RuntimeError):
        ops.expert_mlp(x, x, x[None], x[None], 1, i)
    with pytest.raises(ValueError):
        ops.expert_mlp_workspace(4, 8, 9, 64, 64, "cpu")
