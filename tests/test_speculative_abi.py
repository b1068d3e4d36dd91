"""Host-side refusals of the speculative decoding entry points: checked before any CUDA call, no GPU needed."""

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


def tables(**kw):
    a = dict(t=FAKE, stride=8, rows=4, cols=8, seq_rows=None) | kw
    return ctypes.byref(_lib.PkvTables(*a.values()))


def test_extend_tables():
    def call(t=None, n=4, arrays=FAKE, free=FAKE, num_free=5, head=FAKE, bs=16, total=10, cu=FAKE):
        return L.pkv_extend_tables(t or tables(), n, arrays, arrays, arrays, free, num_free, head, bs, cu, arrays, FAKE, FAKE,
                                   total, arrays, head, None, None)

    assert call(arrays=None) == BAD and call(free=None) == BAD and call(head=None) == BAD and call(cu=None) == BAD
    assert call(n=-1) == BAD and call(bs=0) == BAD and call(num_free=-1) == BAD and call(total=-1) == BAD
    assert call(total=2**31) == BAD and call(tables(rows=3)) == BAD and call(tables(t=None)) == BAD
    assert call(tables(rows=5000), n=4097) == UNSUPPORTED


def test_build_tree_metadata():
    def call(parents=FAKE, cu=FAKE, n=2, total=10, words=1, mask=FAKE):
        return L.pkv_build_tree_metadata(parents, cu, n, FAKE, total, mask, words, FAKE, None, None)

    assert call(parents=None) == BAD and call(cu=None) == BAD and call(mask=None) == BAD and call(n=-1) == BAD
    assert call(total=-1) == BAD and call(words=0) == BAD and call(words=9) == UNSUPPORTED and call(total=0) == OK


def test_rotary_append():
    def call(p=None, layer=0, qkv=FAKE, stride=18 * 64, n=4, hq=14, rotary=64, inter=0, q=FAKE, k=FAKE, slots=None):
        return L.pkv_rotary_append(p or pool(), layer, qkv, stride, n, hq, FAKE, FAKE, rotary, inter, 1.0, q, 896, 64, k, 128, 64,
                                   None, 0, 0, slots, None, None)

    assert call(qkv=None) == BAD and call(q=None) == BAD and call(k=None) == BAD and call(n=-1) == BAD and call(hq=13) == BAD
    assert call(rotary=66) == BAD and call(rotary=0) == BAD and call(rotary=3) == BAD and call(inter=2) == BAD
    assert call(stride=17 * 64) == BAD and call(qkv=FAKE + 1) == BAD
    assert call(layer=2, slots=FAKE) == BAD and call(pool(k=None), slots=FAKE) == BAD
    assert call(pool(dtype=7)) == UNSUPPORTED and call(pool(d=1024), stride=18 * 1024, rotary=1024) == UNSUPPORTED
    assert call(hq=1 << 19, stride=1 << 30) == UNSUPPORTED
    assert call(n=0, qkv=None) == OK


def test_tree_attention():
    need = L.pkv_tree_attention_workspace_bytes(4, 64)
    assert need > 0 and need % 256 == 0
    assert L.pkv_tree_attention_workspace_bytes(4, 96) == 0 and L.pkv_tree_attention_workspace_bytes(1025, 64) == 0
    assert L.pkv_tree_attention_workspace_bytes(0, 64) == 0

    def call(p=None, layer=0, t=None, n=4, cu=FAKE, most=10, total=40, hq=14, out=FAKE, qs=896, k=FAKE, ks=128, mask=FAKE, words=1,
             scale=0.125, ws=FAKE, nbytes=need):
        return L.pkv_tree_attention(p or pool(), layer, t or tables(), n, cu, FAKE, most, total, hq, out, 896, 64, FAKE, qs, 64, k, ks,
                                    64, FAKE, 128, 64, mask, words, scale, ws, nbytes, None, None)

    assert call(cu=None) == BAD and call(out=None) == BAD and call(k=None) == BAD and call(mask=None) == BAD and call(ws=None) == BAD
    assert call(layer=2) == BAD and call(n=-1) == BAD and call(most=65) == BAD and call(words=0) == BAD and call(hq=13) == BAD
    assert call(scale=0.0) == BAD and call(scale=-1.0) == BAD and call(scale=math.nan) == BAD
    assert call(qs=895) == BAD and call(out=FAKE + 2) == BAD and call(k=FAKE + 8) == BAD and call(ks=124) == BAD
    assert call(t=tables(rows=3)) == BAD and call(ws=FAKE + 8) == BAD and call(nbytes=need - 1) == WORKSPACE
    assert call(words=9) == UNSUPPORTED and call(pool(bs=8)) == UNSUPPORTED and call(pool(d=96)) == UNSUPPORTED
    assert call(hq=34) == UNSUPPORTED and call(t=tables(rows=2000), n=1025) == UNSUPPORTED and call(pool(dtype=5)) == UNSUPPORTED
    assert call(n=0) == OK and call(total=0, cu=None) == OK and call(qs=0) == BAD and call(ks=0) == BAD and call(ks=-128) == BAD


def test_accept_tree():
    def call(p=None, t=None, n=4, nodes=FAKE, cu=FAKE, total=40, width=8, outs=FAKE, kv=FAKE):
        return L.pkv_accept_tree(p or pool(), t or tables(), n, nodes, cu, total, nodes, nodes, kv, 5120, 128, 64, kv, 5120, 128, 64,
                                 FAKE, outs, outs, outs, width, outs, None, None)

    assert call(nodes=None) == BAD and call(cu=None) == BAD and call(outs=None) == BAD and call(kv=None) == BAD
    assert call(kv=FAKE + 1) == BAD and call(n=-1) == BAD and call(total=-1) == BAD and call(width=0) == BAD
    assert call(t=tables(rows=3)) == BAD and call(pool(k=None)) == BAD and call(pool(layers=0)) == BAD
    assert call(width=65) == UNSUPPORTED and call(pool(dtype=5)) == UNSUPPORTED and call(n=0) == OK


def test_wrappers_need_cuda_tensors():
    x, i = torch.zeros(1, 1, 64, dtype=torch.float16), torch.zeros(2, dtype=torch.int32)
    p, t = _lib.PkvPool(FAKE, FAKE, 1, 1, 1, 16, 64, 0), _lib.PkvTables(FAKE, 1, 1, 1, None)
    with pytest.raises(RuntimeError):
        ops.tree_attention(p, 0, t, x, x, x, i, i, i.long()[:, None], 1, i)
    with pytest.raises(RuntimeError):
        ops.rotary_append(p, 0, x[0], i.long(), i.double(), 1)
    with pytest.raises(RuntimeError):
        ops.extend_tables(t, i, i, i, i, i, 16, i, i)
    with pytest.raises(RuntimeError):
        ops.build_tree_metadata(i, i, i, i.long()[:, None], i.long())
    with pytest.raises(RuntimeError):
        ops.accept_tree(p, t, i, i, i.long(), i.long(), x, x, i, i, i, i)
