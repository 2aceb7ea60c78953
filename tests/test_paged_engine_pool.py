"""The engine's pool as paged caches: a PagedKV keeps its engine alive, and once the pool has been reserved or grown again the
caches and tables made before are refused instead of reaching memory that is gone.  No GPU: the pool is host memory here, the
library's pool calls are stubs, and a call that is not refused fails on the missing operators."""
import gc
import weakref

import pytest
import torch

from seedplane_amd import paged
from seedplane_amd.qwen_engine import Qwen2Engine

HD, NKV = 64, 2


class _Pool:
    """The pool calls of the library, and nothing else."""
    def sp_engine_kv_reserve(self, *a):
        return 0

    def sp_engine_kv_grow(self, *a):
        return 0


class _Reached(Exception):
    pass


@pytest.fixture
def make_engine(monkeypatch):
    def pages(self, k, v, k_scale=None, v_scale=None):
        self.k, self.v, self.device, self.n_kv_heads, self.head_dim = k, v, k.device, k.shape[1], k.shape[3]

    def reached(*a, **kw):
        raise _Reached
    monkeypatch.setattr(paged.PagedKV, '__init__', pages)
    monkeypatch.setattr(paged, '_call', reached)
    monkeypatch.setattr(Qwen2Engine, '_kv_pool', lambda self, layer: tuple(
        torch.zeros((self._pool_n, NKV, self._pool_slots, HD), dtype=torch.float16) for _ in range(2)))
    monkeypatch.setattr(paged.AttentionPlan, 'workspace_bytes', 0)

    def make():
        eng = Qwen2Engine.__new__(Qwen2Engine)
        eng.lib, eng.h, eng.device = _Pool(), None, torch.device('cpu')
        eng.n_layers, eng.n_kv_heads, eng.head_dim, eng.max_tokens = 2, NKV, HD, 16
        eng.config = {'max_position_embeddings': 4096}
        eng._pool_n = eng._pool_slots = eng._epoch = eng._pool_generation = 0
        eng._free, eng._live = [], weakref.WeakValueDictionary()
        return eng
    return make


@pytest.fixture
def engine(make_engine):
    return make_engine()


def append(kv, table):
    x, i = torch.zeros((3, NKV, HD), dtype=torch.float16), torch.zeros(3, dtype=torch.int32)
    kv.desc, kv.lib, kv._ref = None, type('', (), {'sp_op_paged_append': None}), None
    return kv.append(x, x, i, i, table)


def attend(kv, table):
    plan = paged.AttentionPlan.__new__(paged.AttentionPlan)
    plan.device, plan.n_heads, plan.head_dim, plan.rows, plan.h, plan._ws_addr, plan._scale = kv.device, NKV, HD, 3, None, 0, 1.0
    plan.lib, kv._ref = type('', (), {'sp_op_paged_attention': None}), None
    q, out = (torch.zeros((3, NKV, HD), dtype=torch.float16) for _ in range(2))
    return plan.run(q, kv, table, out=out)


def test_a_paged_cache_keeps_its_engine_alive(make_engine):
    engine = make_engine()
    engine.reserve(2, 64)
    kv, alive = engine.paged_kv(0, 16), weakref.ref(engine)
    del engine
    gc.collect()
    assert alive() is not None
    with pytest.raises(_Reached):
        append(kv, torch.zeros((1, 4), dtype=torch.int32))
    del kv
    gc.collect()
    assert alive() is None


@pytest.mark.parametrize('call', [append, attend])
@pytest.mark.parametrize('change', [
    lambda e: e.new_cache(128),                              # more slots than the pool has
    lambda e: [e.new_cache(32) for _ in range(3)],           # more sequences
    lambda e: e.grow(5, 64), lambda e: e.reserve(2, 64)])
def test_caches_of_an_older_pool_are_refused(engine, change, call):
    engine.reserve(2, 64)
    kv = engine.paged_kv(0, 16)
    rows = torch.zeros((1, 4), dtype=torch.int32)
    with pytest.raises(_Reached):
        call(kv, rows)
    keep = change(engine)
    with pytest.raises(ValueError, match='paged_kv'):
        call(kv, rows)
    with pytest.raises(_Reached):
        call(engine.paged_kv(0, 16), rows)
    del keep


@pytest.mark.parametrize('call', [append, attend])
def test_tables_of_an_older_pool_or_of_other_pages_are_refused(engine, call):
    engine.reserve(2, 64)
    c = engine.new_cache(64)
    table = engine.page_table([c], 16)
    with pytest.raises(_Reached):
        call(engine.paged_kv(1, 16), table)
    with pytest.raises(ValueError, match='page_table'):
        call(engine.paged_kv(1, 32), table)
    engine.grow(2, 128)
    with pytest.raises(ValueError, match='page_table'):
        call(engine.paged_kv(1, 16), table)
    with pytest.raises(_Reached):
        call(engine.paged_kv(1, 16), engine.page_table([c], 16))


def test_a_grow_that_changes_nothing_keeps_them(engine):
    engine.reserve(3, 64)
    kv = engine.paged_kv(0, 16)
    engine.grow(2, 32)
    c = engine.new_cache(64)
    with pytest.raises(_Reached):
        append(kv, engine.page_table([c], 16))
