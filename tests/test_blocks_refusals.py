"""Caches with a scale per block: the C entry points and PagedKV refuse bad arguments before any GPU call (the pointers here are never
dereferenced)."""
import ctypes

import pytest
import torch

from seedplane_amd import _lib
from seedplane_amd.paged import PagedKV

P = 1 << 20
I8, E4M3 = _lib.SP_DT_I8, _lib.SP_DT_E4M3


def cache(dtype=I8, k=P, v=2 * P, ks=3 * P, vs=4 * P, stride=4 * 32 * 64, head=32 * 64, row=64, n=8, page=32, nkv=4, hd=64, block=16):
    return _lib.PagedKVDesc(k, v, ks, vs, stride, head, row, dtype, n, page, nkv, hd, block)


def append(kv=None, rot=64, dtype=_lib.SP_DT_F16, rows=4, heads=8, q=8 * P, k=9 * P, v=10 * P, q_out=12 * P, hd=64, width=4):
    kv = cache() if kv is None else kv
    r = _lib.RotaryDesc(P, rot, 0, 1.0, 0)
    return _lib.load().sp_op_paged_append(ctypes.byref(kv), ctypes.byref(r), dtype, rows, heads, q, 16 * hd, hd, k, 4 * hd, hd, v, 4 * hd, hd,
                                          P, P, P, P, 2, width, q_out, dtype, 8 * hd, hd, None)


def read(kv=None, dtype=_lib.SP_DT_F16, rows=4, seq=P, at=P, table=P, n_seq=2, width=4, k=8 * P, k_row=256, k_head=64, v=9 * P):
    kv = cache() if kv is None else kv
    return _lib.load().sp_op_paged_read(ctypes.byref(kv) if kv else None, dtype, rows, seq, at, table, n_seq, width, k, k_row, k_head, v, 256, 64,
                                        None)


BAD = [dict(ks=None), dict(vs=None), dict(block=0), dict(block=8), dict(block=24), dict(block=-16), dict(page=256, block=256), dict(page=40, block=16),
       dict(dtype=_lib.SP_DT_F16), dict(dtype=_lib.SP_DT_F16, ks=None, vs=None), dict(dtype=5), dict(dtype=E4M3, block=48)]


@pytest.mark.parametrize('kw', BAD)
def test_caches_are_refused_everywhere(kw):
    assert append(cache(**kw)) == _lib.SP_EINVAL and _lib.load().sp_last_error()
    assert read(cache(**kw)) == _lib.SP_EINVAL and _lib.load().sp_last_error()


@pytest.mark.parametrize('kw', [
    dict(kv=cache(vs=3 * P)), dict(kv=cache(vs=3 * P + 64)), dict(kv=cache(ks=P + 64)), dict(kv=cache(vs=2 * P)), dict(k=3 * P),
    dict(v=4 * P - 8), dict(q=3 * P), dict(q_out=4 * P), dict(width=(1 << 25) + 1),
    dict(kv=cache(page=128, block=128, hd=256, row=256, head=128 * 256, stride=4 * 128 * 256), rot=256, hd=256),
    dict(kv=cache(page=128, block=128, hd=512, row=512, head=128 * 512, stride=4 * 128 * 512), rot=64, hd=512, heads=1, q_out=14 * P),
])
def test_append_refusals(kw):
    assert append(**kw) == _lib.SP_EINVAL and _lib.load().sp_last_error()


@pytest.mark.parametrize('kw', [
    dict(kv=False), dict(dtype=E4M3), dict(dtype=I8), dict(rows=-1), dict(n_seq=0), dict(width=0), dict(seq=None), dict(at=None), dict(table=None),
    dict(k=None), dict(v=None), dict(k=9 * P), dict(k=P), dict(v=2 * P), dict(k=3 * P), dict(v=4 * P), dict(k_row=255), dict(k_head=0), dict(k_row=0),
])
def test_read_refusals(kw):
    assert read(**kw) == _lib.SP_EINVAL and _lib.load().sp_last_error()


def test_no_rows_is_no_call():
    assert read(rows=0, seq=None, k=None, v=None) == _lib.SP_OK and append(rows=0) == _lib.SP_OK


def test_python_refusals():
    pool = lambda dtype: torch.zeros((3, 2, 32, 64), dtype=dtype)
    codes, e4m3 = pool(torch.int8), pool(torch.float8_e4m3fn)
    scale = lambda *s: torch.ones(s)
    for k, ks, vs in [(codes, None, None), (codes, scale(2), scale(2)), (codes, scale(3, 2, 2), None), (codes, scale(3, 2, 2), scale(3, 2, 1)),
                      (codes, scale(3, 2, 4), scale(3, 2, 4)), (codes, scale(3, 2, 3), scale(3, 2, 3)), (codes, scale(2, 2, 2), scale(2, 2, 2)),
                      (codes, scale(3, 2, 2).half(), scale(3, 2, 2).half()), (codes, scale(3, 2, 4)[:, :, ::2], scale(3, 2, 4)[:, :, ::2]),
                      (e4m3, scale(3, 2), scale(3, 2)), (pool(torch.float16), scale(3, 2, 2), scale(3, 2, 2))]:
        with pytest.raises(ValueError):
            PagedKV(k, k.clone(), ks, vs)
    for block in (0, -16, 12):
        with pytest.raises((ValueError, RuntimeError)):
            PagedKV.allocate(3, 32, 2, 64, torch.int8, scale_block=block, device='cuda:0')
