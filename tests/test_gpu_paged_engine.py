"""The engine's own K/V as paged caches: a document that the engine prefilled once is the shared prefix of a batch."""
import pytest
import torch

from conftest import small_cfg
from paged_ref import attend64
from seedplane_amd.paged import AttentionPlan
from seedplane_amd.qwen_engine import Qwen2Engine
from seedplane_amd.synth import make_weights

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def engine():
    cfg, w = make_weights(small_cfg(), 'q8', seed=3)
    eng = Qwen2Engine(config=cfg, tensors=w, max_tokens=16)
    eng.reserve(6, 192)
    return eng


def test_the_engines_pool_is_the_prefix_of_a_batch(gpu_device, engine):
    g = torch.Generator().manual_seed(0)
    ids = lambda n: torch.randint(0, 1000, (n,), generator=g).tolist()
    doc = engine.new_cache(192)
    engine.prefill([ids(96)], [doc])
    own = [engine.new_cache(64) for _ in range(4)]
    counts = [5, 33, 64, 1]
    engine.prefill([ids(n) for n in counts], own)
    page, P = 32, 96
    table = torch.cat([engine.page_table([doc], page)[:, :P // page].expand(4, -1), engine.page_table(own, page)], 1).contiguous()
    kv_lens = [P + n for n in counts]
    nh, nkv, hd = engine.n_heads, engine.n_kv_heads, engine.head_dim
    plan = AttentionPlan(nh, nkv, hd, 8, 4).set([1, 2, 4, 1], kv_lens, [(4, P)])
    q = torch.randn((8, nh, hd), generator=g).half().to(gpu_device)
    for layer in (0, -1):
        kv = engine.paged_kv(layer, page)
        k, v = (torch.zeros((kv.n_pages, nkv, page, hd), dtype=torch.float16) for _ in range(2))
        for c, rows in [(doc, engine.page_table([doc], page)[0])] + list(zip(own, engine.page_table(own, page))):
            for pool, copy in ((k, c.keys[layer]), (v, c.values[layer])):      # [1, capacity, kv_heads, head_dim]
                for i in range(-(-c.length // page)):
                    part = copy[0, i * page:(i + 1) * page].permute(1, 0, 2).cpu()
                    pool[int(rows[i]), :, :part.shape[1]] = part
        want, _, bound = attend64(q, k, v, table, [1, 2, 4, 1], kv_lens, hd ** -0.5)
        got = plan.run(q, kv, table).double().cpu()
        assert ((got - want).abs() <= bound).all()


def test_whole_rings_as_pages_and_refusals(gpu_device, engine):
    c = engine.new_cache(100)
    engine.prefill([[1, 2, 3, 4, 5]], [c])
    kv, table = engine.paged_kv(0), engine.page_table([c])
    assert kv.page_size == 192 and table.shape == (1, 1) and torch.equal(kv.k[int(table), :, :5].permute(1, 0, 2), c.keys[0][0, :5])
    with pytest.raises(ValueError):
        engine.paged_kv(0, 100)
    with pytest.raises(IndexError):
        engine.paged_kv(7)
    wrapped = engine.new_cache(4096, window=64)
    wrapped.length = 193
    with pytest.raises(ValueError):
        engine.page_table([wrapped])


def test_a_pool_that_grows_or_whose_engine_is_let_go(gpu_device):
    """After the pool has grown by itself the older pages are refused and new ones read the same positions; the pages outlive the
    program's own reference to the engine."""
    cfg, w = make_weights(small_cfg(), 'q8', seed=3)
    eng = Qwen2Engine(config=cfg, tensors=w, max_tokens=16)
    eng.reserve(1, 64)
    doc = eng.new_cache(64)
    eng.prefill([[7, 8, 9, 10, 11] * 6], [doc])
    nh, nkv, hd = eng.n_heads, eng.n_kv_heads, eng.head_dim
    plan = AttentionPlan(nh, nkv, hd, 2, 1).set([2], [30])
    q = torch.randn((2, nh, hd), generator=torch.Generator().manual_seed(1)).half().to(gpu_device)
    old, old_table = eng.paged_kv(1, 16), eng.page_table([doc], 16)
    want = plan.run(q, old, old_table)
    other = eng.new_cache(128)                                 # more slots and more sequences than the pool has
    new = torch.zeros((1, nkv, hd), dtype=torch.float16, device=gpu_device)
    at = torch.zeros(1, dtype=torch.int32, device=gpu_device)
    kv, table = eng.paged_kv(1, 16), eng.page_table([doc], 16)
    for bad in (lambda: plan.run(q, old, old_table), lambda: plan.run(q, old, table), lambda: plan.run(q, kv, old_table),
                lambda: old.append(new, new, at, at, old_table)):
        with pytest.raises(ValueError):
            bad()
    assert torch.equal(plan.run(q, kv, table), want)
    del eng, other, doc
    assert torch.equal(plan.run(q, kv, table), want)
