"""Beam search on the engine (generate_beams), and a serving loop of the operators around it: beams of several requests over a paged
cache of 8 bits, forked, appended and read together."""
import math

import numpy as np
import pytest
import torch

from blocks_ref import attend_blocks64, dense64
from conftest import small_cfg
from seedplane_amd.beam import beam_select
from seedplane_amd.paged import AttentionPlan, PagedKV, Rotary
from seedplane_amd.pages import PagePool
from seedplane_amd.qwen_engine import Qwen2Engine
from seedplane_amd.synth import make_weights

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def engine():
    cfg, w = make_weights(small_cfg(), 'q8', seed=3)
    return Qwen2Engine(config=cfg, tensors=w, max_tokens=16)


def _search(engine, prompt, K, steps, eos, penalty):
    """Beam search as its definition has it: every step's logits from a fresh pass over each beam's whole text."""
    live, done = [([], 0.0)], []
    for step in range(steps):
        every = []
        for b, (ids, total) in enumerate(live):
            logp = torch.log_softmax(engine.forward(prompt + ids)[0][0].double().cpu(), -1)
            top = torch.sort(logp, descending=True, stable=True).indices[:2 * K].tolist()
            every += [(total + float(logp[t]), b, t) for t in top]
        every = sorted(every, key=lambda e: (-e[0], e[1], e[2]))[:K * (1 if eos is None else 2)]
        done += [(live[b][0] + [t], s / (step + 1) ** penalty) for s, b, t in every if t == eos]
        done = sorted(done, key=lambda d: -d[1])[:K]
        live = [(live[b][0] + [t], s) for s, b, t in every if t != eos][:K]
        now = [s / (step + 1) ** penalty for _, s in live]
        if step + 1 == steps or (len(done) == K and max(now) <= done[-1][1]):
            done += [(ids, s / (step + 1) ** penalty) for ids, s in live]
            break
    return sorted(done, key=lambda d: -d[1])[:K]


def _score(engine, prompt, ids, penalty):
    """Of a continuation, from one pass over all of it."""
    logits = engine.forward(prompt + ids[:-1], all_logits=True)[0].double().cpu()
    logp = torch.log_softmax(logits[len(prompt) - 1:], -1)
    return sum(float(logp[i, t]) for i, t in enumerate(ids)) / len(ids) ** penalty


@pytest.mark.parametrize('n,K,steps,penalty,use_eos', [(5, 4, 6, 1.0, True), (70, 3, 5, 0.0, False), (1, 1, 4, 1.0, True), (33, 8, 12, 0.6, True)])
def test_beams_of_an_engine(gpu_device, engine, n, K, steps, penalty, use_eos):
    """The continuations' scores are those of a pass over their text; no continuation that the definition's search finds is better
    than the best by more than the passes' own differences (fp16 activations: logits within 2e-2 of each other here, so a sum of
    `steps` log probabilities within steps x 4e-2), and with these the search itself may differ."""
    prompt = torch.randint(0, 1000, (n,), generator=torch.Generator().manual_seed(n)).tolist()
    eos = int(engine.forward(prompt)[0][0].topk(2).indices[1]) if use_eos else None
    got = engine.generate_beams(prompt, beams=K, max_new_tokens=steps, eos_token_id=eos, length_penalty=penalty)
    want = _search(engine, prompt, K, steps, eos, penalty)
    assert 1 <= len(got) <= K and [s for _, s in got] == sorted((s for _, s in got), reverse=True)
    assert len(set(tuple(i) for i, _ in got)) == len(got)
    for ids, s in got:
        assert 1 <= len(ids) <= steps and (eos not in ids[:-1]) and (len(ids) == steps or ids[-1] == eos)
        assert abs(s - _score(engine, prompt, ids, penalty)) <= 4e-2 * len(ids) / len(ids) ** penalty
    assert got[0][1] >= want[0][1] - 4e-2 * steps
    if K == 1 and eos is None:
        assert got[0][0] == list(engine.generate(prompt, steps))


def test_beams_of_an_engine_refusals(gpu_device, engine):
    for kw in (dict(beams=0), dict(beams=17), dict(max_new_tokens=0), dict(max_new_tokens=5000), dict(beams=33, eos_token_id=1)):
        with pytest.raises(ValueError):
            engine.generate_beams([1, 2, 3], **kw)
    with pytest.raises(ValueError):
        engine.generate_beams([])


def test_requests_with_beams_over_pages(gpu_device):
    """Two requests of three beams: prompts appended once and forked, then steps of append, attention, selection and fork, requests
    replaced half way.  Every step's attention against the 64-bit form over what the cache holds, and what each beam holds against
    what was appended along its ancestors."""
    g = torch.Generator().manual_seed(31)
    B, K, nh, nkv, hd, page, V = 2, 3, 6, 2, 64, 16, 500
    S, layers = B * K, 2
    caches = [PagedKV.allocate(60, page, nkv, hd, torch.int8, scale_block=16) for _ in range(layers)]
    pool = PagePool(caches, S, 8)
    rotary, plan = Rotary(hd), AttentionPlan(nh, nkv, hd, 64, S)
    ints = lambda x: torch.as_tensor(x, dtype=torch.int32).to(gpu_device)
    texts = [[] for _ in range(S)]                            # of each sequence: the values appended at its positions (layer 0)
    scores = torch.full((B, K), -math.inf, device=gpu_device)

    def admit(b, n):
        """A prompt of n positions for request b, in its first beam."""
        x = torch.randn((n, 2 * nkv, hd), generator=g).half().to(gpu_device)
        counts = np.zeros(S, int)
        counts[b * K] = n
        pool.grow(ints(counts))
        for kv in caches:
            kv.append(x[:, :nkv], x[:, nkv:], ints([b * K] * n), ints(range(n)), pool.table, rotary=rotary)
        texts[b * K] = [x[i, nkv:].cpu() for i in range(n)]
        scores[b, 0], scores[b, 1:] = 0, -math.inf
    admit(0, 21)
    admit(1, 32)
    for step in range(10):
        if step == 5:                                        # the second request ends, another begins
            pool.free(ints(range(K, 2 * K)))
            for s in range(K, 2 * K):
                texts[s] = []
            pool.compact()
            admit(1, 45)
        lens = pool.lengths.tolist()
        step_select = beam_select(torch.randn((S, V), generator=g).to(gpu_device) * 3, scores, eos=7)
        parents = step_select.next_rows.view(-1)
        pool.fork(parents)
        rows = parents.tolist()
        assert pool.lengths.tolist() == [lens[p] if p >= 0 else 0 for p in rows]
        texts = [list(texts[p]) if p >= 0 else [] for p in rows]
        scores = step_select.next_scores
        # one position more for every beam
        x = torch.randn((S, nh + 2 * nkv, hd), generator=g).half().to(gpu_device)
        at = pool.lengths.clone()
        pool.grow(ints([1] * S))
        for kv in caches:
            q = kv.append(x[:, nh:nh + nkv], x[:, nh + nkv:], ints(range(S)), at, pool.table, rotary=rotary, q=x[:, :nh])
        for s in range(S):
            texts[s].append(x[s, nh + nkv:].cpu())
        lens = pool.lengths.tolist()
        shared = [min(int(n) for n in lens[b * K:(b + 1) * K]) - 1 for b in range(B)]
        same = []
        table = pool.table.cpu()
        for b in range(B):
            part = table[b * K:(b + 1) * K]
            common = 0
            while (common + 1) * page <= shared[b] and (part[:, common] == part[0, common]).all():
                common += 1
            same.append((K, common * page))
        plan.set([1] * S, lens, same)
        kv = caches[0]
        out = plan.run(q, kv, pool.table)
        want, _, bound = attend_blocks64(q, kv.k, kv.k_scale, kv.v, kv.v_scale, pool.table, [1] * S, lens, hd ** -0.5)
        assert float(((out.double().cpu() - want).abs() - bound).max()) <= 0
        held = dense64(kv.v, kv.v_scale)
        for s in range(S):
            _, v = kv.read(ints([s] * lens[s]), ints(range(lens[s])), pool.table, dtype=torch.float32)
            text = torch.stack(texts[s]).double()
            assert torch.equal(v.double().cpu().float(), torch.stack([held[int(table[s, p // page]), :, p % page] for p in range(lens[s])]).float())
            # a value was rounded once when it came and at most once more for each later position of its block
            limit = torch.stack([kv.v_scale[int(table[s, p // page]), :, 0].double().cpu() for p in range(lens[s])])
            assert float(((v.double().cpu() - text).abs() - limit[..., None] * 0.5 * 16).max()) <= 0
        count = torch.zeros(60, dtype=torch.int64).index_add_(0, table[table >= 0].long(), torch.ones(int((table >= 0).sum()), dtype=torch.int64))
        assert pool.holders.tolist() == count.tolist() and int(pool.missing) == 0
        for kv0, kv1 in [(caches[0], caches[1])]:
            used = pool.holders > 0
            assert torch.equal(kv0.k_scale[used], kv1.k_scale[used]) and int(used.sum()) <= 60
