"""Pools whose pages lie on each other (an engine's rings seen as pages: page e's second head is another page's first) only copy: the calls
that give pages to sequences are refused, in C and in Python.  No GPU: the pointers here are never dereferenced."""
import ctypes
import weakref

import pytest
import torch

from seedplane_amd import _lib, paged, pages
from seedplane_amd.qwen_engine import Qwen2Engine

P = 1 << 20
HD, NKV, SLOTS, PAGE = 64, 2, 128, 64


def desc(n_pages, nkv, page, page_stride, head_stride, row_stride, hd=HD):
    return _lib.PagePoolDesc(P, None, P, P, P, P, P, page_stride, head_stride, row_stride, 6, _lib.SP_DT_F16, n_pages, page, nkv, hd, 0, 5, 7, 1)


@pytest.mark.parametrize('sizes', [
    (6, 2, 64, 64 * HD, 128 * HD, HD),                       # rings of 128 slots, two heads each
    (3, 2, 64, 64 * HD, 128 * HD, HD),                       # just one page too many
    (2, 2, 16, 16 * HD, 16 * HD, HD),                        # pages and heads at one stride
    (4, 3, 16, 3 * 16 * HD - 1, 16 * HD, HD), (4, 3, 16, 3 * 16 * HD, 16 * HD - 1, HD), (4, 3, 16, 3 * HD, HD, 2 * HD),
    (2, 1, 4, HD + 8, HD, HD), (1 << 30, 2, 1 << 20, 1 << 40, 1 << 60, 1 << 41)])
def test_overlapping_pages_are_refused(sizes):
    lib, ref = _lib.load(), ctypes.byref(desc(*sizes))
    for rc in (lib.sp_op_pages_fork(ref, P, None), lib.sp_op_pages_grow(ref, P, None), lib.sp_op_pages_free(ref, 2, P, None),
               lib.sp_op_pages_free(ref, 0, None, None), lib.sp_op_pages_compact(ref, None, None)):
        assert rc == _lib.SP_EINVAL and b'each other' in lib.sp_last_error()
    assert lib.sp_op_pages_copy(ref, 0, None, None, None) == _lib.SP_OK


@pytest.mark.parametrize('sizes', [
    (2, 2, 64, 64 * HD, 128 * HD, HD),                       # pages within a head, as many as a ring has
    (6, 2, 16, 2 * 16 * HD, 16 * HD, HD), (6, 2, 16, 2 * 16 * HD, HD, 2 * HD),     # heads first, rows first
    (6, 2, 16, 3 * 17 * 80, 17 * 80, 80), (1, 2, 16, 0, HD, 2 * HD), (6, 1, 16, 16 * HD, 0, HD), (6, 2, 1, 2 * HD, HD, 0)])
def test_pages_apart_are_not_refused(sizes):
    assert _lib.load().sp_op_pages_free(ctypes.byref(desc(*sizes)), 0, None, None) == _lib.SP_OK


class _Reached(Exception):
    pass


def _engine_pool(monkeypatch, nkv):
    """A pool over an engine's rings in host memory; calls that are not refused raise _Reached."""
    def init(self, k, v, k_scale=None, v_scale=None):
        self.k, self.v, self.k_scale, self.v_scale, self.scale_block = k, v, k_scale, v_scale, 0
        self.device, self.dtype, self.lib = k.device, k.dtype, _lib.load()
        self.n_pages, self.n_kv_heads, self.page_size, self.head_dim = k.shape

    def reached(*a, **kw):
        raise _Reached
    monkeypatch.setattr(paged.PagedKV, '__init__', init)
    monkeypatch.setattr(pages, '_call', reached)
    monkeypatch.setattr(pages, '_raw_stream', lambda device: 0)
    eng = Qwen2Engine.__new__(Qwen2Engine)
    eng.device, eng.n_layers, eng.n_kv_heads, eng.head_dim = torch.device('cpu'), 2, nkv, HD
    eng._pool_n, eng._pool_slots, eng._epoch, eng._pool_generation, eng._live = 2, SLOTS, 0, 1, weakref.WeakValueDictionary()
    rings = [tuple(torch.randn((2, nkv, SLOTS, HD)).half() for _ in range(2)) for _ in range(2)]
    eng._kv_pool = lambda layer: rings[layer]
    return eng, pages.PagePool([eng.paged_kv(layer, PAGE) for layer in range(2)], 3, 2)


@pytest.mark.parametrize('nkv', [1, 2])
def test_a_pool_over_an_engines_rings_only_copies(monkeypatch, nkv):
    eng, pool = _engine_pool(monkeypatch, nkv)
    v = pool.caches[0].v
    if nkv == 2:
        assert torch.equal(v[SLOTS // PAGE, 0], v[0, 1])      # one memory, two pages
    ints = lambda *x: torch.tensor(x, dtype=torch.int32)
    for call in (lambda: pool.fork(ints(0, 1, 2)), lambda: pool.grow(ints(1, 1, 1)), lambda: pool.free(ints(0)), lambda: pool.compact()):
        with pytest.raises(ValueError, match='engine'):
            call()
    with pytest.raises(_Reached):
        pool.copy(ints(0), ints(1))
