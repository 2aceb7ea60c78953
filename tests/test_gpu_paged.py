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
