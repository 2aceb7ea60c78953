"""The loop of selection, forks, growth, appends and attention where beams end on the way: an ended beam holds no page and no position, its row of
the batch writes nothing and reads nothing, until a fork makes it another beam's child."""
import math

import pytest
import torch

from blocks_ref import attend_blocks64
from seedplane_amd.beam import beam_select
from seedplane_amd.paged import AttentionPlan, PagedKV, Rotary
from seedplane_amd.pages import PagePool

pytestmark = pytest.mark.gpu


def test_ended_beams_take_nothing(gpu_device):
    g = torch.Generator().manual_seed(77)
    B, K, nh, nkv, hd, page, V, n_pages = 2, 3, 6, 2, 64, 16, 40, 50
    S = B * K
    caches = [PagedKV.allocate(n_pages, page, nkv, hd, torch.int8, scale_block=16) for _ in range(2)]
    pool, rotary, plan = PagePool(caches, S, 8), Rotary(hd), AttentionPlan(nh, nkv, hd, S, S)
    index = torch.arange(S, dtype=torch.int32, device=gpu_device)
    prompt = torch.zeros(S, dtype=torch.int32, device=gpu_device)
    prompt[0], prompt[K] = 20, 32
    pool.grow(prompt)
    scores = torch.full((B, K), -math.inf, device=gpu_device)
    scores[:, 0] = 0
    for s, n in ((0, 20), (K, 32)):
        x = torch.randn((n, 2 * nkv, hd), generator=g).half().to(gpu_device)
        for kv in caches:
            kv.append(x[:, :nkv], x[:, nkv:], torch.full((n,), s, dtype=torch.int32, device=gpu_device),
                      torch.arange(n, dtype=torch.int32, device=gpu_device), pool.table, rotary=rotary)
    ended = 0
    for step in range(12):
        logits = torch.randn((S, V), generator=g) * 2
        logits[:, torch.randperm(V, generator=g)[:V - (1, 2, 5)[step % 3]]] = -math.inf      # a grammar that allows few tokens
        best = beam_select(logits.to(gpu_device), scores, eos=[])
        scores = best.next_scores
        parents = best.next_rows.view(-1)
        live = parents >= 0
        pool.fork(parents)
        at = pool.lengths.clone()
        pool.grow(live.int())
        seq = torch.where(live, index, -1)
        x = torch.randn((S, nh + 2 * nkv, hd), generator=g).half().to(gpu_device)
        before = [(kv.k.clone(), kv.k_scale.clone()) for kv in caches]
        for kv in caches:
            q = kv.append(x[:, nh:nh + nkv], x[:, nh + nkv:], seq, at, pool.table, rotary=rotary, q=x[:, :nh])
        lens = pool.lengths.tolist()
        alive = live.tolist()
        ended += S - sum(alive)
        assert all((n > 0) == a for n, a in zip(lens, alive))
        table = pool.table.cpu()
        assert all(int((row >= 0).sum()) == -(-n // page) for row, n in zip(table, lens))
        held = torch.bincount(table[table >= 0].long(), minlength=n_pages)
        assert pool.holders.tolist() == held.tolist() and int(pool.missing) == 0
        for kv, (k, ks) in zip(caches, before):              # an append changes the pages of live beams' last positions alone
            last = [int(table[s, (lens[s] - 1) // page]) for s in range(S) if alive[s]]
            other = [e for e in range(n_pages) if e not in last]
            assert torch.equal(kv.k[other], k[other]) and torch.equal(kv.k_scale[other], ks[other])
        plan.set([1] * S, lens)
        out = plan.run(q, caches[1], pool.table)
        kv = caches[1]
        want, _, bound = attend_blocks64(q, kv.k, kv.k_scale, kv.v, kv.v_scale, pool.table, [1] * S, lens, hd ** -0.5)
        assert float(((out.double().cpu() - want).abs() - bound).max()) <= 0
        assert all(not out[s].any() for s in range(S) if not alive[s])
    assert ended >= 4
