"""Paged K/V operators on the GPU against plain 64-bit forms: rotation, append, attention with shared prefixes, and a run of
them together.  Tolerances: tests/paged_ref.py derives them beside the forms."""
import math

import numpy as np
import pytest
import torch

from paged_ref import HALF, TINY, attend64, paged_batch, rotate64, rotate_bound
from seedplane_amd import paged
from seedplane_amd.paged import AttentionPlan, PagedKV, Rotary

pytestmark = pytest.mark.gpu

F32, F16, BF16, E4M3 = torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn
YARN = {'rope_type': 'yarn', 'factor': 4.0, 'original_max_position_embeddings': 32768}


def _within(got, want, bound):
    got = got.double().cpu()
    assert torch.isfinite(got).all() or not torch.isfinite(want).all()
    over = ((got - want).abs() - bound)
    at = int(over.argmax())
    assert float(over.max()) <= 0, (at, float(got.flatten()[at]), float(want.flatten()[at]), float(bound.flatten()[at]))


# ------------------------------------------------------------------------------------------------ rotate
@pytest.mark.parametrize('dtype', [F32, F16, BF16])
@pytest.mark.parametrize('rows,heads,hd,rot,layout,scaling', [
    (1, 1, 64, 64, 'half', None), (16, 18, 64, 64, 'half', None), (777, 3, 128, 64, 'interleaved', YARN),
    (33, 32, 128, 128, 'interleaved', None), (5, 7, 80, 32, 'half', YARN), (9, 2, 6, 2, 'half', None),
    (9, 3, 10, 6, 'interleaved', None), (300, 40, 256, 256, 'half', None)])
def test_rotate(gpu_device, dtype, rows, heads, hd, rot, layout, scaling):
    print(f'rotate {dtype} {rows} {heads} {hd} {rot} {layout}', flush=True)
    g = torch.Generator().manual_seed(rows * 7 + hd)
    r = Rotary(hd, theta=1e6, rot_dim=rot, layout=layout, scaling=scaling)
    x = torch.randn((rows, heads, hd), generator=g).to(dtype)
    pos = torch.randint(-1000, 2 ** 31 - 1, (rows,), generator=g, dtype=torch.int64).to(torch.int32)
    pos[0] = 0
    want = rotate64(x, pos, r.inv_freq, r.factor, rot, layout)
    # positions of 2^31: a 64-bit angle of 2e9 rad is off by 2^-22 of a radian's 2^-2 at most, i.e. by 2^31 x 2^-53
    bound = rotate_bound(x, rot, layout, r.factor, dtype, want) + 2.0 ** -20 * x.double().abs().amax()
    got = r.apply(x.to(gpu_device), pos.to(gpu_device))
    _within(got, want, bound)
    assert torch.equal(got.cpu()[..., rot:], x[..., rot:])
    # a view with wider rows and heads, into a view, and in place
    wide = torch.full((rows, heads + 2, hd + 8), 7.0, dtype=dtype, device=gpu_device)
    wide[:, 1:1 + heads, :hd] = x.to(gpu_device)
    view = wide[:, 1:1 + heads, :hd]
    out = torch.full((rows, heads, 2 * hd), 9.0, dtype=dtype, device=gpu_device)
    r.apply(view, pos.to(gpu_device), out=out[..., :hd])
    assert torch.equal(out[..., :hd], got) and (out[..., hd:] == 9).all()
    r.apply(view, pos.to(gpu_device), out=view)
    assert torch.equal(view, got)
    assert (wide[:, 0] == 7).all() and (wide[:, heads + 1:] == 7).all() and (wide[..., hd:] == 7).all()


def test_rotate_far_positions_and_back(gpu_device):
    """Angles of far positions keep their accuracy, and negated positions undo the rotation (and are its gradient)."""
    r = Rotary(128, theta=1e6)
    x = torch.randn((64, 4, 128), generator=torch.Generator().manual_seed(1)).to(gpu_device)
    pos = torch.arange(1000000, 1000064, dtype=torch.int32, device=gpu_device)
    y = r.apply(x, pos)
    _within(y, rotate64(x, pos, r.inv_freq, 1.0, 128, 'half'),
            rotate_bound(x, 128, 'half', 1.0, F32, x.double().cpu() * 0) + 2.0 ** -22 * x.double().cpu().abs().amax())
    back = r.apply(y, -pos)
    assert float((back - x).abs().max()) <= 4 * 2.0 ** -21 * 2 * float(x.abs().max())
    # gradient: <R x, w> has the gradient R^T w = rotation of w by -pos; against a difference in the direction of d
    w, d = (torch.randn(x.shape, generator=torch.Generator().manual_seed(s)).to(gpu_device) for s in (2, 3))
    grad = r.apply(w, -pos).double()
    diff = ((r.apply(x + d, pos).double() - r.apply(x - d, pos).double()) * w.double()).sum() / 2
    size = float((w.double().abs() * d.double().abs()).sum()) + float((w.double().abs() * x.double().abs()).sum())
    assert abs(float((grad * d.double()).sum() - diff)) <= 2.0 ** -19 * size


def test_rotate_empty_and_views_on_unaligned_memory(gpu_device):
    r = Rotary(64, rot_dim=32)
    none = torch.empty((0, 3, 64), device=gpu_device)
    assert r.apply(none, torch.empty(0, dtype=torch.int32, device=gpu_device)).shape == (0, 3, 64)
    buf = torch.randn(1 + 10 * 3 * 64, generator=torch.Generator().manual_seed(0)).half().to(gpu_device)
    x = buf[1:].view(10, 3, 64)                            # 2-byte aligned: values one by one
    pos = torch.arange(10, dtype=torch.int32, device=gpu_device)
    assert torch.equal(r.apply(x, pos), r.apply(x.clone(), pos))


# ------------------------------------------------------------------------------------------------ append
def _append_case(g, dev, rows, dtype, cache, nh, nkv, hd, page, n_seq, far, bad=True):
    width = -(-far // page)
    n_pages = n_seq * width + 2
    table = torch.randperm(n_pages, generator=g)[:n_seq * width].to(torch.int32).view(n_seq, width)
    spots = torch.randperm(n_seq * far, generator=g)[:rows]
    seq, at = (spots // far).to(torch.int32), (spots % far).to(torch.int32)
    if bad and rows >= 8:
        seq[1], at[2], seq[3], at[4] = -1, -1, n_seq, width * page
        table[int(seq[5]), int(at[5]) // page] = n_pages       # entries outside the pool
        table[int(seq[6]), int(at[6]) // page] = -3
    heads = torch.randn((rows, nh + 2 * nkv, hd), generator=g).to(dtype)
    e4m3 = cache == E4M3
    scales = tuple((torch.rand(nkv, generator=g) + 0.5).mul(0.008).to(dev) for _ in range(2)) if e4m3 else (None, None)
    pools = [(torch.randn((n_pages, nkv, page, hd), generator=g)).to(cache).to(dev) for _ in range(2)]
    return table, seq, at, heads, scales, pools


@pytest.mark.parametrize('dtype,cache', [(F16, F16), (BF16, BF16), (F32, F16), (F32, E4M3), (BF16, E4M3), (F16, BF16)])
@pytest.mark.parametrize('rows,nh,nkv,hd,rot,page,layout', [
    (16, 12, 2, 128, 128, 16, 'half'), (1, 14, 2, 64, 64, 1, 'half'), (200, 28, 4, 128, 64, 24, 'interleaved'),
    (11, 3, 3, 40, 12, 5, 'half'), (64, 0, 8, 64, 0, 128, 'half')])
def test_append(gpu_device, dtype, cache, rows, nh, nkv, hd, rot, page, layout):
    print(f'append {dtype} {cache} {rows} {nh} {nkv} {hd} {rot} {page} {layout}', flush=True)
    g = torch.Generator().manual_seed(rows + hd + page)
    table, seq, at, heads, scales, pools = _append_case(g, gpu_device, rows, dtype, cache, nh, nkv, hd, page, 7, 300)
    n_pages = pools[0].shape[0]
    before = [p.clone() for p in pools]
    kv = PagedKV(*pools, *scales)
    rotary = Rotary(hd, theta=1e6, rot_dim=rot, layout=layout, scaling=YARN) if rot else None
    turn = torch.randint(0, 100000, (rows,), generator=g).to(torch.int32)
    d = heads.to(gpu_device)
    q, k, v = d[:, :nh], d[:, nh:nh + nkv], d[:, nh + nkv:]
    q_out = torch.full((rows, nh, hd), 5.0, dtype=dtype, device=gpu_device) if nh else None
    got = kv.append(k, v, seq.to(gpu_device), at.to(gpu_device), table.to(gpu_device), rotary=rotary, q=q if nh else None,
                    q_out=q_out, rotary_pos=turn.to(gpu_device))
    assert got is q_out
    if rot:
        both = rotate64(heads[:, :nh + nkv], turn, rotary.inv_freq, rotary.factor, rot, layout)
        args = (rot, layout, rotary.factor)
    else:
        both = heads[:, :nh + nkv].double()
    want = [p.double().cpu() for p in before]
    bound = [torch.zeros_like(w) for w in want]
    alive = []
    for r in range(rows):
        s, p = int(seq[r]), int(at[r])
        if not (0 <= s < table.shape[0] and 0 <= p // page < table.shape[1] and p >= 0):
            continue
        e = int(table[s, p // page])
        if not 0 <= e < n_pages:
            continue
        alive.append(r)
        for i, new in enumerate((both[r, nh:], heads[r, nh + nkv:].double())):
            err = torch.zeros_like(new)
            if i == 0 and rot:
                raw = heads[r:r + 1, nh:nh + nkv]
                err = rotate_bound(raw, *args, F32, both[r:r + 1, nh:])[0]
            if cache == E4M3:
                sc = scales[i].cpu().double()[:, None]
                new, err = (new / sc).clamp(-448, 448), err / sc + (new / sc).abs() * 2.0 ** -23
            want[i][e, :, p % page] = new
            bound[i][e, :, p % page] = err + (new.abs() + err) * HALF[cache] + TINY[cache]
    for pool, w, b, old in zip(pools, want, bound, before):
        _within(pool.float(), w, b)
        same = b == 0
        assert torch.equal(pool.cpu().view(torch.uint8 if cache == E4M3 else torch.int16)[same],
                           old.cpu().view(torch.uint8 if cache == E4M3 else torch.int16)[same])
    if nh:
        alive = torch.tensor(alive)
        wq = both[:, :nh][alive]
        b = rotate_bound(heads[:, :nh][alive], *args, dtype, wq) if rot else torch.zeros_like(wq)
        _within(q_out[alive.to(gpu_device)], wq, b)
        dead = [r for r in range(rows) if r not in set(alive.tolist())]
        assert (q_out[dead] == 5).all()


def test_append_saturates_and_keeps_nan(gpu_device):
    kv = PagedKV.allocate(2, 4, 1, 64, E4M3, torch.ones(1, device=gpu_device), torch.ones(1, device=gpu_device))
    x = torch.zeros((1, 1, 64), device=gpu_device)
    x[0, 0, :6] = torch.tensor([1e9, -1e9, math.inf, -math.inf, math.nan, 460.0])
    i = torch.zeros(1, dtype=torch.int32, device=gpu_device)
    kv.append(x, x, i, i, i.view(1, 1))
    for pool in (kv.k, kv.v):
        row = pool[0, 0, 0].float().tolist()
        assert row[:4] == [448, -448, 448, -448] and math.isnan(row[4]) and row[5] == 448 and row[6:] == [0] * 58


def test_append_in_place_queries_and_default_output(gpu_device):
    g = torch.Generator().manual_seed(3)
    table, seq, at, heads, _, pools = _append_case(g, gpu_device, 20, F16, F16, 4, 2, 64, 16, 3, 50)
    kv, r = PagedKV(*pools), Rotary(64)
    d = heads.to(gpu_device)
    call = lambda q, **kw: kv.append(d[:, 4:6], d[:, 6:], seq.to(gpu_device), at.to(gpu_device), table.to(gpu_device), rotary=r, q=q, **kw)
    fresh = call(d[:, :4])
    def lives(s, p):                                       # (other rows may lie on the pages that rows 5 and 6 lose)
        return 0 <= s < 3 and 0 <= p < 4 * 16 and 0 <= int(table[s, p // 16]) < pools[0].shape[0]
    dead = [i for i in range(20) if not lives(int(seq[i]), int(at[i]))]
    assert set(range(1, 7)) <= set(dead) and len(dead) < 20
    assert (fresh[dead] == 0).all()
    own = d[:, :4].clone()
    assert call(own, q_out=own) is own
    live = [i for i in range(20) if i not in dead]
    assert torch.equal(own[live], fresh[live]) and torch.equal(own[dead], d[:, :4][dead])


# ------------------------------------------------------------------------------------------------ attention
def _attend(dev, q_lens, kv_lens, groups, nh, nkv, hd, page, dtype, cache, seed=0, lse=True, scale=None, **kw):
    g = torch.Generator().manual_seed(seed)
    behind = kw.pop('rows_behind', 3)
    q, k, v, table, scales = paged_batch(g, q_lens, kv_lens, groups, nh, nkv, hd, page, dtype, cache, dev, rows_behind=behind, **kw)
    kv = PagedKV(k, v, *scales)
    plan = AttentionPlan(nh, nkv, hd, max_rows=max(1, sum(q_lens)), max_seqs=len(q_lens))
    plan.set(q_lens, kv_lens, groups)
    out = torch.full(q.shape, 3.0, dtype=dtype, device=dev)
    ls = torch.full(q.shape[:2], 3.0, device=dev) if lse else None
    plan.run(q, kv, table, out=out, lse=ls, scale=scale)
    torch.cuda.synchronize()
    n = sum(q_lens)
    want, wl, bound = attend64(q[:n], k, v, table, q_lens, kv_lens, scale or hd ** -0.5, *scales)
    _within(out[:n], want, bound)
    assert (out[n:] == 3).all()
    if lse:
        got = ls[:n].double().cpu()
        assert torch.equal(got == -math.inf, wl == -math.inf) and (ls[n:] == 3).all()
        seen = wl > -math.inf
        assert float((got - wl)[seen].abs().max() if seen.any() else 0) <= 2.0 ** -15 * (1 + float(wl[seen].abs().max() if seen.any() else 0))
    return plan, q, kv, table, out


TYPES = [(F16, F16), (BF16, BF16), (F16, E4M3), (BF16, E4M3)]


@pytest.mark.parametrize('dtype,cache', TYPES)
@pytest.mark.parametrize('hd', [64, 128])
@pytest.mark.parametrize('q_lens,kv_lens,groups,nh,nkv,page', [
    ([1], [1], None, 2, 1, 16),
    ([1], [733], None, 14, 2, 16),
    ([1] * 5, [5, 64, 65, 1, 300], None, 4, 4, 7),
    ([1] * 16, [2048 // 8 + i * 9 for i in range(16)], [(16, 256)], 12, 2, 16),
    ([1] * 40, [515 + i for i in range(40)], [(20, 512), (20, 480)], 28, 4, 32),
    ([3, 0, 1, 9], [200, 90, 150, 160], [(4, 80)], 12, 2, 16),
    ([40, 7], [140, 107], [(2, 96)], 28, 4, 24),
    ([2, 5, 1], [0, 3, 0], None, 6, 2, 16),
    ([33, 70], [33, 70], None, 8, 1, 64),
    ([1, 1], [1300, 1301], [(2, 1299)], 32, 1, 1),
])
def test_attention(gpu_device, dtype, cache, hd, q_lens, kv_lens, groups, nh, nkv, page):
    print(f'attend {dtype} {cache} {hd} {q_lens} {kv_lens} {groups} {nh} {nkv} {page}', flush=True)
    _attend(gpu_device, q_lens, kv_lens, groups, nh, nkv, hd, page, dtype, cache, seed=len(q_lens) + hd)


@pytest.mark.parametrize('seed', range(24))
def test_random_batches(gpu_device, seed):
    """Head counts, page sizes, groups (of sequences without queries too), drafts, prompts and lone tokens drawn together."""
    rng = np.random.default_rng(1000 + seed)
    nkv = int(rng.choice([1, 2, 3, 4]))
    nh = nkv * int(rng.choice([1, 2, 5, 6, 7, 16, 32]))
    hd, page = int(rng.choice([64, 128])), int(rng.choice([1, 8, 16, 20, 64]))
    dtype, cache = TYPES[seed % 4]
    q_lens, kv_lens, groups = [], [], []
    for _ in range(rng.integers(1, 4)):
        size, shared = int(rng.integers(1, 7)), int(rng.integers(0, 700)) // page * page
        for _ in range(size):
            q = int(rng.choice([0, 1, 1, 1, 2, 5, 9, 33, 70]))
            q_lens.append(q)
            kv_lens.append(shared + int(rng.integers(0, 260)))     # (a draft may begin within the shared positions, or before any)
        groups.append((size, shared))
    print(f'random {seed}: {nh}/{nkv} heads of {hd}, pages of {page}, {dtype} {cache}, {q_lens} {kv_lens} {groups}', flush=True)
    _attend(gpu_device, q_lens, kv_lens, groups, nh, nkv, hd, page, dtype, cache, seed=seed)


def test_layouts_of_the_pool(gpu_device):
    """Heads before rows, rows before heads, keys and values in one allocation, one page, one head: append and attention."""
    nkv, hd, page, n, L = 2, 64, 16, 12, 150
    g = torch.Generator().manual_seed(6)
    x = torch.randn((L, 4 + 2 * nkv, hd), generator=g).half().to(gpu_device)
    at = torch.arange(L, dtype=torch.int32, device=gpu_device)
    table = torch.randperm(n, generator=g).int().view(1, n).to(gpu_device)
    plan = AttentionPlan(4, nkv, hd, 9, 1).set([9], [L])
    zeros = lambda *s: torch.zeros(s, dtype=F16, device=gpu_device)
    nhd, both, apart = zeros(2, n, page, nkv, hd), zeros(n, 2, nkv, page, hd), zeros(2, n, nkv + 1, page + 3, 2 * hd)
    outs, pools = [], []
    for kv in (PagedKV.allocate(n, page, nkv, hd), PagedKV(nhd[0].transpose(1, 2), nhd[1].transpose(1, 2)), PagedKV(both[:, 0], both[:, 1]),
               PagedKV(apart[0, :, :nkv, :page, :hd], apart[1, :, :nkv, :page, :hd])):
        kv.append(x[:, 4:4 + nkv], x[:, 4 + nkv:], torch.zeros_like(at), at, table)
        outs.append(plan.run(x[-9:, :4], kv, table))
        pools.append((kv.k.clone(), kv.v.clone()))
    assert all(torch.equal(o, outs[0]) for o in outs) and all(torch.equal(a, b) for p in pools for a, b in zip(p, pools[0]))
    assert (apart[:, :, nkv:] == 0).all() and (apart[:, :, :, page:] == 0).all() and (apart[..., hd:] == 0).all()
    _within(outs[0], *attend64(x[-9:, :4], *pools[0], table, [9], [L], 0.125)[::2])
    one = PagedKV(zeros(1, 1, 200, hd), zeros(1, 1, 200, hd))
    t1 = torch.zeros((1, 1), dtype=torch.int32, device=gpu_device)
    one.append(x[:, 4:5], x[:, 6:7], torch.zeros_like(at), at, t1)
    got = AttentionPlan(2, 1, hd, 9, 1).set([9], [L]).run(x[-9:, :2], one, t1)
    _within(got, *attend64(x[-9:, :2], one.k, one.v, t1, [9], [L], 0.125)[::2])


def test_attention_views_pages_apart_scale_and_no_lse(gpu_device):
    """q and out as views of wider rows, pages further apart than their size, another scale, no lse."""
    q_lens, kv_lens, groups = [1, 4, 1], [90, 100, 70], [(3, 64)]
    plan, q, kv, table, want = _attend(gpu_device, q_lens, kv_lens, groups, 12, 2, 128, 16, F16, F16, seed=5, scale=0.2,
                                       stride=2 * 2 * 16 * 128, rows_behind=0)
    wide = torch.full((6, 40, 136), 2.0, dtype=F16, device=gpu_device)
    wide[:, 3:15, :128] = q
    out = torch.full((6, 13, 160), 4.0, dtype=F16, device=gpu_device)
    got = plan.run(wide[:, 3:15, :128], kv, table, out=out[:, 1:, 8:136], scale=0.2)
    assert torch.equal(got, want) and (out[:, 0] == 4).all() and (out[..., :8] == 4).all() and (out[..., 136:] == 4).all()
    assert torch.equal(plan.run(q, kv, table, scale=0.2), want)


@pytest.mark.parametrize('fill', [math.inf, -math.inf, 1e4])
@pytest.mark.parametrize('cache', [F16, BF16])
def test_what_the_pool_holds_elsewhere_does_not_matter(gpu_device, fill, cache):
    _attend(gpu_device, [1, 20, 3], [33, 47, 3], None, 14, 2, 64, 16, cache, cache, seed=9, fill=fill)


@pytest.mark.parametrize('dtype,cache', [(F16, F16), (BF16, E4M3)])
def test_entries_outside_the_pool_hide_their_positions(gpu_device, dtype, cache):
    """Of a shared prefix, of a sequence's own positions, and all of a sequence's: zeros and lse -inf where nothing is left."""
    g = torch.Generator().manual_seed(11)
    q_lens, kv_lens, groups = [1, 1, 20, 2, 1], [300, 280, 290, 20, 16], [(3, 256), (1, 0), (1, 0)]
    q, k, v, table, scales = paged_batch(g, q_lens, kv_lens, groups, 14, 2, 128, 16, dtype, cache, gpu_device)
    bad = k.shape[0]
    table[:3, 5] = bad
    table[:3, 15] = -1
    table[1, 17] = 1 << 30
    table[2, 18] = -(1 << 31)
    table[3] = -7
    kv = PagedKV(k, v, *scales)
    plan = AttentionPlan(14, 2, 128, max_rows=25, max_seqs=5).set(q_lens, kv_lens, groups)
    lse = torch.zeros(25, 14, device=gpu_device)
    out = plan.run(q, kv, table, lse=lse)
    want, wl, bound = attend64(q, k, v, table, q_lens, kv_lens, 128 ** -0.5, *scales)
    _within(out, want, bound)
    assert torch.equal(lse.cpu() == -math.inf, wl == -math.inf) and (out[22:24] == 0).all() and (lse[22:24] == -math.inf).all()


def test_long_contexts(gpu_device):
    """Parts of many row tables, more parts than the join's waves hold at once, a prefix of an odd page size."""
    _attend(gpu_device, [1], [40000], None, 2, 1, 64, 16, F16, F16, seed=1)
    _attend(gpu_device, [1, 1, 1], [9003, 9100, 9001], [(3, 9000)], 28, 4, 128, 24, BF16, BF16, seed=2)
    _attend(gpu_device, [1] * 24, [2500 + 3 * i for i in range(24)], [(24, 2450)], 8, 2, 64, 49, BF16, E4M3, seed=3)
    _attend(gpu_device, [130], [5000], None, 4, 4, 64, 128, F16, F16, seed=4)


def test_peaked_and_extreme_scores(gpu_device):
    """Scores of hundreds (one weight is all), large values next to the type's limit, and a late maximum after many flat ones."""
    g = torch.Generator().manual_seed(2)
    q, k, v, table, _ = paged_batch(g, [1, 30], [700, 730], None, 8, 2, 64, 16, F16, F16, gpu_device)
    q *= 40
    v *= 3000
    k[int(table[0, 40])] *= 5
    kv = PagedKV(k, v)
    plan = AttentionPlan(8, 2, 64, 31, 2).set([1, 30], [700, 730])
    _within(plan.run(q, kv, table), *attend64(q, k, v, table, [1, 30], [700, 730], 0.125)[::2])


@pytest.mark.parametrize('dtype,cache', TYPES)
@pytest.mark.parametrize('q_lens,kv_lens,groups,nh,nkv,hd', [
    ([1, 3, 5], [40, 300, 2900], None, 12, 2, 128),
    ([40, 9], [140, 4109], None, 8, 2, 64),
    ([130, 20], [130, 700], None, 28, 4, 128),
    ([6, 6], [518, 530], [(2, 512)], 14, 2, 64),
])
def test_infinities_and_nans_reach_only_the_rows_and_columns_that_see_them(gpu_device, dtype, cache, q_lens, kv_lens, groups, nh, nkv, hd):
    """A later token's values may be anything: earlier rows do not see them, other columns do not meet them."""
    g = torch.Generator().manual_seed(9)
    q, k, v, table, scales = paged_batch(g, q_lens, kv_lens, groups, nh, nkv, hd, 16, dtype, cache, gpu_device)
    scale = hd ** -0.5
    want, _, bound = attend64(q, k, v, table, q_lens, kv_lens, scale, *scales)
    plan = AttentionPlan(nh, nkv, hd, sum(q_lens), len(q_lens)).set(q_lens, kv_lens, groups)
    inf = math.inf if cache != E4M3 else math.nan
    r0 = 0
    for s, (nq, n) in enumerate(zip(q_lens, kv_lens)):
        back, last = max(0, nq // 2), r0 + nq - 1                # the token seen from row last - back on, and the newest
        mid, end = n - 1 - back, n - 1
        page, slot = int(table[s, mid // 16]), mid % 16
        v[page, :, slot, 3] = inf
        v[page, :, slot, 7] = math.nan
        v[page, :, slot, 9] = inf
        want[last - back:last + 1, :, 3] = inf
        want[last - back:last + 1, :, 7] = math.nan
        want[last - back:last + 1, :, 9] = inf
        if back:
            v[int(table[s, end // 16]), :, end % 16, 9] = -inf
            want[last, :, 9] = math.nan
            v[int(table[s, end // 16]), :, end % 16, hd - 1] = -inf
            want[last, :, hd - 1] = -inf
        r0 += nq
    out = plan.run(q, PagedKV(k, v, *scales), table).double().cpu()
    assert torch.equal(out.isnan(), want.isnan())
    whole = want.isfinite()
    assert torch.equal(out[~whole & ~want.isnan()], want[~whole & ~want.isnan()])
    assert ((out - want).abs() <= bound)[whole].all()


def test_a_nan_key_reaches_the_rows_that_see_it(gpu_device):
    """Outputs and lse of the rows that see it, in one item and in parts."""
    g = torch.Generator().manual_seed(10)
    q_lens, kv_lens = [1, 4, 2], [60, 300, 5000]
    q, k, v, table, _ = paged_batch(g, q_lens, kv_lens, None, 8, 2, 64, 16, F16, F16, gpu_device)
    for s, n in enumerate(kv_lens):
        k[int(table[s, (n - 1) // 16]), :, (n - 1) % 16] = math.nan
    plan = AttentionPlan(8, 2, 64, 7, 3).set(q_lens, kv_lens)
    lse = torch.zeros(q.shape[:2], device=gpu_device)
    out = plan.run(q, PagedKV(k, v), table, lse=lse)
    seen = torch.tensor([1, 0, 0, 0, 1, 0, 1], dtype=torch.bool)
    assert torch.equal(out.isnan().all(-1).all(-1).cpu(), seen) and torch.equal(out.isnan().any(-1).any(-1).cpu(), seen)
    assert torch.equal(lse.isnan().all(-1).cpu(), seen) and torch.equal(lse.isnan().any(-1).cpu(), seen)


def test_a_table_dropped_after_its_call_on_another_stream(gpu_device):
    """Memory of a rotary table that goes out of use while another stream still reads it is not given out again."""
    x = torch.randn((2048, 32, 128), device=gpu_device)
    pos = torch.arange(2048, dtype=torch.int32, device=gpu_device)
    want = Rotary(128, theta=1e6).apply(x, pos)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = x
        for _ in range(20):
            y = y * 1.0                                        # work ahead of the call
    r = Rotary(128, theta=1e6)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = r.apply(y, pos)
    del r
    for _ in range(50):
        torch.full((64,), math.nan, dtype=torch.float64, device=gpu_device)
    side.synchronize()
    assert torch.equal(got, want)


def test_values_near_the_least_and_the_greatest(gpu_device):
    """Contexts read in parts whose values are all subnormal, all zero, or large."""
    g = torch.Generator().manual_seed(11)
    q, k, v, table, _ = paged_batch(g, [1, 1, 1], [9000, 9000, 9000], None, 4, 2, 64, 16, BF16, BF16, gpu_device)
    for s, size in enumerate((2.0 ** -128, 0.0, 2.0 ** 90)):
        pages = table[s, :-(-9000 // 16)].long()
        v[pages] = (v[pages].float() * size).to(BF16)
    plan = AttentionPlan(4, 2, 64, 3, 3).set([1] * 3, [9000] * 3)
    _within(plan.run(q, PagedKV(k, v), table), *attend64(q, k, v, table, [1] * 3, [9000] * 3, 0.125)[::2])


def test_offsets_past_32_bits(gpu_device):
    """Pages whose elements lie beyond 2^32 of the pool's start: append and attention."""
    free, _ = torch.cuda.mem_get_info(gpu_device)
    nkv, hd, page = 2, 128, 16
    n, stride = 40, 1 << 27                                  # 40 pages, 2^27 elements apart: 10 GiB each for k and v
    if free < 26 << 30:
        pytest.skip('needs 26 GiB of free memory')
    pools = [torch.empty((n, stride), dtype=F16, device=gpu_device)[:, :nkv * page * hd].view(n, nkv, page, hd) for _ in range(2)]
    kv = PagedKV(*pools)
    L = 4 * page
    table = torch.tensor([[39, 33, 36, 38]], dtype=torch.int32, device=gpu_device)
    g = torch.Generator().manual_seed(0)
    x = torch.randn((L, 3 * nkv, hd), generator=g).half().to(gpu_device)
    at = torch.arange(L, dtype=torch.int32, device=gpu_device)
    kv.append(x[:, :nkv], x[:, nkv:2 * nkv], torch.zeros_like(at), at, table)
    for i, p in enumerate(table[0].tolist()):
        assert torch.equal(pools[0][p], x[i * page:(i + 1) * page, :nkv].permute(1, 0, 2))
        assert torch.equal(pools[1][p], x[i * page:(i + 1) * page, nkv:2 * nkv].permute(1, 0, 2))
    plan = AttentionPlan(nkv, nkv, hd, L, 1).set([L], [L])
    q = x[:, 2 * nkv:].contiguous()
    small = [torch.zeros((40, nkv, page, hd), dtype=F16) for _ in range(2)]
    for s, p in zip(small, pools):
        s[table[0].cpu().long()] = p[table[0].long()].cpu()
    want, _, bound = attend64(q, small[0], small[1], table, [L], [L], hd ** -0.5)
    _within(plan.run(q, kv, table), want, bound)


def test_results_repeat_bit_for_bit_and_do_not_depend_on_the_stream(gpu_device):
    plan, q, kv, table, out = _attend(gpu_device, [1] * 12, [700 + 31 * i for i in range(12)], [(12, 640)], 28, 4, 128, 16, BF16, BF16)
    for _ in range(3):
        assert torch.equal(plan.run(q[:12], kv, table), out[:12])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = plan.run(q[:12], kv, table, workspace=torch.empty(plan.workspace_bytes, dtype=torch.uint8, device=gpu_device))
        b = Rotary(128).apply(q[:12], torch.arange(12, dtype=torch.int32, device=gpu_device))
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a, out[:12])
    assert torch.equal(b, Rotary(128).apply(q[:12], torch.arange(12, dtype=torch.int32, device=gpu_device)))


def test_two_plans_on_two_streams(gpu_device):
    """Plans have workspaces of their own: batches that run side by side do not meet."""
    runs = []
    for seed, n in ((0, 9), (1, 5)):
        runs.append(_attend(gpu_device, [1] * n, [900 + 50 * i for i in range(n)], [(n, 896)], 12, 2, 128, 16, F16, F16, seed=seed, lse=False))
    streams = [torch.cuda.Stream() for _ in runs]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(10):
        for i, ((plan, q, kv, table, _), s) in enumerate(zip(runs, streams)):
            with torch.cuda.stream(s):
                outs[i].append(plan.run(q, kv, table))
    torch.cuda.synchronize()
    for i, (_, q, _, _, want) in enumerate(runs):
        n = q.shape[0] - 3
        assert all(torch.equal(o[:n], want[:n]) and (o[n:] == 0).all() for o in outs[i])


def test_captured_step_follows_later_lengths(gpu_device):
    """Append and attention captured once; lengths, tables and positions change between replays, eager work in between."""
    nh, nkv, hd, page, B, width = 12, 2, 128, 16, 6, 64
    g = torch.Generator().manual_seed(4)
    n_pages = B * width
    kv = PagedKV(*[torch.randn((n_pages, nkv, page, hd), generator=g).half().to(gpu_device) for _ in range(2)])
    table = torch.randperm(n_pages, generator=g).int().view(B, width).to(gpu_device)
    table[:, :8] = table[0, :8]                               # 128 common positions
    r = Rotary(hd, theta=1e6)
    x = torch.randn((B, nh + 2 * nkv, hd), generator=g).half().to(gpu_device)
    seq = torch.arange(B, dtype=torch.int32, device=gpu_device)
    at = torch.zeros(B, dtype=torch.int32, device=gpu_device)
    qr, out = (torch.zeros((B, nh, hd), dtype=F16, device=gpu_device) for _ in range(2))
    plan = AttentionPlan(nh, nkv, hd, B, B)
    lens = [200 + 17 * i for i in range(B)]

    def step():
        kv.append(x[:, nh:nh + nkv], x[:, nh + nkv:], seq, at, table, rotary=r, q=x[:, :nh], q_out=qr)
        plan.run(qr, kv, table, out=out)

    def place(groups):
        at.copy_(torch.tensor(lens, dtype=torch.int32) - 1)
        plan.set([1] * B, lens, groups)
    place([(B, 128)])
    step()                                                    # (warm)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(5):
        lens = [n + 90 * (i % 3) + 1 for n in lens]
        place([(B, 128)] if i % 2 == 0 else None)
        x.copy_(torch.randn(x.shape, generator=g).half())
        graph.replay()
        got = out.clone()
        torch.cuda.synchronize()
        step()
        assert torch.equal(got, out), i
        want, _, bound = attend64(qr, kv.k, kv.v, table, [1] * B, lens, hd ** -0.5)
        _within(got, want, bound)


def test_a_step_captured_before_any_request(gpu_device):
    """A call captured while the plan holds no queries serves the batches set later."""
    g = torch.Generator().manual_seed(8)
    q, k, v, table, _ = paged_batch(g, [1, 2], [700, 90], None, 8, 2, 64, 16, BF16, BF16, gpu_device, rows_behind=1)
    kv = PagedKV(k, v)
    plan = AttentionPlan(8, 2, 64, 4, 2).set([0, 0], [0, 0])
    out = torch.full_like(q, 3.0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.run(q, kv, table, out=out)
    graph.replay()
    torch.cuda.synchronize()
    assert (out == 3).all()
    for lens in ([1, 2], [1, 0], [0, 2]):
        out.fill_(3.0)
        plan.set(lens, [700, 90])
        graph.replay()
        got, n = out.clone(), sum(lens)
        want, _, bound = attend64(q[:n], k, v, table, lens, [700, 90], 0.125)
        _within(got[:n], want, bound)
        assert (got[n:] == 3).all()


def test_set_is_refused_in_a_capture(gpu_device):
    from seedplane_amd._lib import SeedPlaneError
    plan = AttentionPlan(2, 1, 64, 4, 4).set([1], [1])
    y = torch.zeros(1, device=gpu_device)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y += 1
        with pytest.raises(SeedPlaneError):
            plan.set([1], [2])
    graph.replay()
    torch.cuda.synchronize()


def test_many_sets_in_flight(gpu_device):
    """A plan set again and again without waiting: every run sees the lengths set before it."""
    plan, q, kv, table, _ = _attend(gpu_device, [1] * 4, [1000] * 4, None, 4, 2, 64, 16, F16, F16, rows_behind=0)
    wants = {}
    for n in (1000, 3, 517):
        plan.set([1] * 4, [n] * 4)
        wants[n] = plan.run(q, kv, table)
    torch.cuda.synchronize()
    outs = []
    for i in range(60):
        n = (1000, 3, 517)[i % 3]
        plan.set([1] * 4, [n] * 4)
        outs.append((n, plan.run(q, kv, table)))
    torch.cuda.synchronize()
    assert all(torch.equal(o, wants[n]) for n, o in outs)


@pytest.mark.parametrize('dtype,cache', [(F16, F16), (BF16, BF16), (BF16, E4M3)])
def test_a_conversation_as_a_server_runs_it(gpu_device, dtype, cache):
    """One system prompt prefilled once, requests' prompts on top of it, then decode steps and a draft of several tokens:
    positions, pages and sharing as a server keeps them; every step against attention over the tokens so far."""
    nh, nkv, hd, page, B, P = 14, 2, 64, 16, 5, 70            # 70 shared tokens: 4 whole pages and 6 positions of each one's own
    g = torch.Generator().manual_seed(8)
    e4m3 = cache == E4M3
    scales = [torch.full((nkv,), 0.01, device=gpu_device) for _ in range(2)] if e4m3 else [None, None]
    kv = PagedKV.allocate(200, page, nkv, hd, cache, *scales)
    r = Rotary(hd, theta=1e4, scaling={'rope_type': 'linear', 'factor': 2.0})
    plan = AttentionPlan(nh, nkv, hd, max_rows=256, max_seqs=B)
    free = list(range(199, -1, -1))
    shared = [free.pop() for _ in range(P // page)]
    table = np.full((B, 20), -1, np.int32)
    table[:, :len(shared)] = shared
    lens = [0] * B
    hist = [[torch.zeros((0, nkv, hd), dtype=torch.float64) for _ in range(2)] for _ in range(B)]
    head = torch.randn((P, nh + 2 * nkv, hd), generator=g).to(dtype)

    def step(counts, rows, groups):
        for s, n in enumerate(counts):
            for p in range(lens[s] // page, -(-(lens[s] + n) // page)):
                if table[s, p] < 0:
                    table[s, p] = free.pop()
        dev = lambda a: torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(gpu_device)
        seq, at = np.repeat(np.arange(B), counts), np.concatenate([np.arange(lens[s], lens[s] + n) for s, n in enumerate(counts)])
        x, t = rows.to(gpu_device), dev(table)
        q = kv.append(x[:, nh:nh + nkv], x[:, nh + nkv:], dev(seq), dev(at), t, rotary=r, q=x[:, :nh])
        for s, n in enumerate(counts):
            lens[s] += n
        kv_lens = [lens[s] if n else 0 for s, n in enumerate(counts)]
        plan.set(counts, kv_lens, groups)
        out = plan.run(q, kv, t)
        want, _, bound = attend64(q, kv.k, kv.v, t, counts, kv_lens, hd ** -0.5, *(scales if e4m3 else ()))
        _within(out, want, bound)
        # and against the tokens themselves, rotated in 64 bits and rounded to the cache
        turned = rotate64(rows[:, :nh + nkv], torch.from_numpy(at.astype(np.int32)), r.inv_freq, r.factor, hd, 'half')
        i = 0
        for s, n in enumerate(counts):
            for j, new in enumerate((turned[i:i + n, nh:], rows[i:i + n, nh + nkv:].double())):
                if e4m3:
                    new = (new / 0.01).clamp(-448, 448).float().to(E4M3).double() * 0.01
                else:
                    new = new.to(dtype).double()
                hist[s][j] = torch.cat([hist[s][j], new])
            for a in range(n):
                m = lens[s] - n + a + 1
                k, v = (h[:m].repeat_interleave(nh // nkv, 1) for h in hist[s])
                w = torch.softmax((turned[i + a, :nh].to(dtype).double()[None] * k).sum(-1) * hd ** -0.5, 0)
                ref = (w[..., None] * v).sum(0)
                # roundings of the cache that fall on the other side: a step of the cache's type on single keys
                assert float((out[i + a].double().cpu() - ref).abs().max()) <= float(bound[i + a].max()) + 4 * HALF[cache]
            i += n

    # the system prompt goes through sequence 0's table; the others' copies of its last 6 tokens come with their own prompts
    step([P, 0, 0, 0, 0], head, None)
    for s in range(1, B):
        lens[s] = len(shared) * page
        hist[s] = [h[:lens[s]].clone() for h in hist[0]]
    counts = [11, 20, 7, 33, 9]
    rows = torch.cat([torch.cat([head[len(shared) * page:] if s else head[:0], torch.randn((n - (6 if s else 0), nh + 2 * nkv, hd),
                                                                                          generator=g).to(dtype)]) for s, n in enumerate(counts)])
    step(counts, rows, [(B, len(shared) * page)])
    for _ in range(4):
        step([1] * B, torch.randn((B, nh + 2 * nkv, hd), generator=g).to(dtype), [(B, len(shared) * page)])
    step([4, 1, 0, 3, 5], torch.randn((13, nh + 2 * nkv, hd), generator=g).to(dtype), [(2, 64), (3, 64)])


# ------------------------------------------------------------------------------------------------ refusals of the Python layer
def test_python_refusals(gpu_device):
    kv = PagedKV.allocate(4, 16, 2, 64)
    plan = AttentionPlan(4, 2, 64, 8, 4).set([1, 1], [5, 9])
    t = torch.zeros((2, 3), dtype=torch.int32, device=gpu_device)
    q = torch.zeros((2, 4, 64), dtype=F16, device=gpu_device)
    i = torch.zeros(2, dtype=torch.int32, device=gpu_device)
    r = Rotary(64)
    plan.run(q, kv, t)

    def bad(f, kind=ValueError):
        with pytest.raises(kind):
            f()
    bad(lambda: plan.run(q.float(), kv, t))
    bad(lambda: plan.run(q.bfloat16(), kv, t))                   # not the cache's type
    bad(lambda: plan.run(q[:1], kv, t))                          # fewer rows than the plan
    bad(lambda: plan.run(q[:, :2], kv, t))
    bad(lambda: plan.run(q.cpu(), kv, t))
    bad(lambda: plan.run(q, kv, t.long()))
    bad(lambda: plan.run(q, kv, t[:1]))                          # a table of fewer sequences
    bad(lambda: plan.run(q, kv, t[:, ::2]))
    bad(lambda: plan.run(q, kv, t, out=q))
    bad(lambda: plan.run(q, kv, t, out=q.float()))
    bad(lambda: plan.run(q, kv, t, scale=0.0))
    bad(lambda: plan.run(q, kv, t, scale=math.nan))
    bad(lambda: plan.run(q, kv, t, lse=torch.zeros(2, 4, dtype=F16, device=gpu_device)))
    bad(lambda: plan.run(q, kv, t, workspace=torch.zeros(8, dtype=torch.uint8, device=gpu_device)))
    bad(lambda: plan.run(q, PagedKV.allocate(4, 16, 4, 64), t))
    bad(lambda: plan.set([1] * 5, [1] * 5))
    bad(lambda: plan.set([9], [9]))
    bad(lambda: plan.set([1, 1], [5]))
    bad(lambda: plan.set([1, 1], [5, 9], [(1, 5)]))
    bad(lambda: plan.set([1, 1], [5, 9], []))
    bad(lambda: plan.set([1, 1], [5, 49]) and plan.run(q, kv, t))        # longer than the table
    bad(lambda: AttentionPlan(4, 2, 64, 8, 4).run(q, kv, t), RuntimeError)   # no lengths yet
    bad(lambda: AttentionPlan(4, 2, 80, 8, 4))
    bad(lambda: AttentionPlan(4, 2, 64, 8, 4, device='cpu'))
    odd = torch.zeros(2 * 4 * 64 + 1, dtype=F16, device=gpu_device)[1:].view(2, 4, 64)
    plan.set([1, 1], [5, 9])
    bad(lambda: plan.run(odd, kv, t))                            # not aligned to 16 bytes
    bad(lambda: r.apply(q, i.long()))
    bad(lambda: r.apply(q, i[:1]))
    bad(lambda: r.apply(q.half()[:, :, :32], i))
    bad(lambda: r.apply(q, i, out=q[:1]))
    bad(lambda: r.apply(q, i, out=q.float()))
    buf = torch.zeros(3, 4, 64, dtype=F16, device=gpu_device)
    bad(lambda: r.apply(buf[:2], i, out=buf[1:]))
    bad(lambda: r.apply(q, i, out=buf[:1].expand(2, 4, 64)))
    bad(lambda: Rotary(64, layout='other'))
    bad(lambda: Rotary(64, rot_dim=128))
    k = torch.zeros((2, 2, 64), dtype=F16, device=gpu_device)
    app = lambda **kw: kv.append(**{**dict(k=k, v=k, seq=i, pos=i, table=t, rotary=r, q=q), **kw})
    assert app().shape == q.shape
    bad(lambda: app(v=k.float()))
    bad(lambda: app(k=k[:, :1]))
    bad(lambda: app(seq=i[:1]))
    bad(lambda: app(pos=i.long()))
    bad(lambda: app(table=t.view(-1)))
    bad(lambda: app(q=q[:1]))
    bad(lambda: app(q=None, q_out=q))
    bad(lambda: app(q_out=q[:1]))
    bad(lambda: app(q_out=torch.cat([q, q])[1:3], q=torch.cat([q, q])[:2].float()))
    bad(lambda: app(rotary=Rotary(128)))
    z = torch.zeros((4, 2, 16, 64), dtype=F16, device=gpu_device)
    bad(lambda: PagedKV(z, z.float()))
    bad(lambda: PagedKV(z.float(), z.float()))
    bad(lambda: PagedKV(z.transpose(2, 3), z.transpose(2, 3)))
    bad(lambda: PagedKV(z, z.transpose(1, 2).contiguous().transpose(1, 2)))
    bad(lambda: PagedKV(z[:1].expand(4, 2, 16, 64), z))
    bad(lambda: PagedKV(z, z, k_scale=torch.ones(2, device=gpu_device)))
    bad(lambda: PagedKV(z.to(E4M3), z.to(E4M3)))
    bad(lambda: PagedKV(z.cpu(), z.cpu()))
    torch.cuda.synchronize()
