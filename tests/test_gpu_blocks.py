"""Paged caches with a scale per block of positions and head, on the GPU against plain 64-bit forms: append, read, attention, and a
run of them together.  Tolerances: tests/blocks_ref.py derives them beside the forms."""
import math

import numpy as np
import pytest
import torch

from blocks_ref import MOST, append64, attend_blocks64, coded, dense64
from paged_ref import HALF, TINY, paged_batch, rotate64, rotate_bound
from seedplane_amd.paged import AttentionPlan, PagedKV, Rotary

pytestmark = pytest.mark.gpu

F32, F16, BF16, I8, E4M3 = torch.float32, torch.float16, torch.bfloat16, torch.int8, torch.float8_e4m3fn


def _within(got, want, bound):
    got = got.double().cpu()
    here = ~want.isnan()
    over = ((got - want).abs() - bound)[here]
    assert not over.numel() or float(over.max()) <= 0, (float(over.max()), float(((got - want).abs() / bound)[here].nan_to_num().max()))


def _int(x, dev='cuda'):
    return torch.as_tensor(x, dtype=torch.int32).to(dev)


# ------------------------------------------------------------------------------------------------ append and read
def _cache(g, dev, n_pages, nkv, page, hd, cache, block):
    x = [torch.randn((n_pages, nkv, page, hd), generator=g) * (0.5 + torch.rand((n_pages, nkv, page, 1), generator=g)) for _ in range(2)]
    (k, ks), (v, vs) = (coded(t, cache, block) for t in x)
    return PagedKV(k.to(dev), v.to(dev), ks.to(dev), vs.to(dev))


def _check_append(kv, before, new, seq, at, table):
    """The cache against append64 of what it held; new: keys, values in 64 bits with bounds of their own."""
    for (codes, scale), (x, err), pool, sc in zip(before, new, (kv.k, kv.v), (kv.k_scale, kv.v_scale)):
        val, want, bound = append64(codes, scale, x, seq, at, table, kv.page_size)
        # (errors of the new values reach the scale by the largest of them and codes by themselves; then everything moves with the scale)
        far = float(err.max())
        _within(sc, want, want * 2.0 ** -21 + far / MOST[codes.dtype])
        _within(torch.from_numpy(dense64(pool, sc).numpy()), val, bound * (1 + 2.0 ** -20) + 4 * far + (bound > 0) * val.abs() * 2.0 ** -20)
        same = (bound == 0).all(-1)                           # rows that nothing touches keep their bits
        old, now = codes.cpu().view(torch.uint8), pool.cpu().view(torch.uint8)
        assert torch.equal(now[same], old[same])


@pytest.mark.parametrize('dtype', [F32, F16, BF16])
@pytest.mark.parametrize('cache', [I8, E4M3])
@pytest.mark.parametrize('rows,nh,nkv,hd,rot,page,block,layout,order', [
    (16, 12, 2, 128, 128, 16, 16, 'half', 'alone'), (1, 14, 2, 64, 64, 32, 32, 'half', 'alone'),
    (200, 28, 4, 128, 64, 48, 16, 'interleaved', 'runs'), (150, 3, 3, 40, 12, 32, 16, 'half', 'any'),
    (64, 0, 8, 64, 0, 128, 128, 'half', 'runs'), (700, 4, 1, 128, 128, 64, 64, 'half', 'any'), (300, 2, 2, 36, 36, 16, 16, 'interleaved', 'runs')])
def test_append(gpu_device, dtype, cache, rows, nh, nkv, hd, rot, page, block, layout, order):
    print(f'append blocks {dtype} {cache} {rows} {nh} {nkv} {hd} {rot} {page} {block} {order}', flush=True)
    g = torch.Generator().manual_seed(rows + hd + page)
    n_seq, far = (7, 300) if order != 'alone' else (rows, 300)
    width = -(-far // page)
    n_pages = n_seq * width + 2
    table = torch.randperm(n_pages, generator=g)[:n_seq * width].to(torch.int32).view(n_seq, width)
    if order == 'alone':
        seq, at = torch.arange(rows), torch.randint(0, far, (rows,), generator=g)
    else:
        spots = torch.randperm(n_seq * far, generator=g)[:rows]
        if order == 'runs':
            spots = spots.sort().values
        seq, at = spots // far, spots % far
    seq, at = seq.to(torch.int32), at.to(torch.int32)
    if rows >= 8:
        seq[1], at[2], seq[3], at[4] = -1, -1, n_seq, width * page
        table[int(seq[5]), int(at[5]) // page] = n_pages
        table[int(seq[6]), int(at[6]) // page] = -3
    kv = _cache(g, gpu_device, n_pages, nkv, page, hd, cache, block)
    before = [(kv.k.clone(), kv.k_scale.clone()), (kv.v.clone(), kv.v_scale.clone())]
    heads = (torch.randn((rows, nh + 2 * nkv, hd), generator=g) * torch.rand((rows, 1, 1), generator=g) * 2).to(dtype)
    turn = torch.randint(0, 100000, (rows,), generator=g).to(torch.int32)
    rotary = Rotary(hd, theta=1e6, rot_dim=rot, layout=layout) if rot else None
    d = heads.to(gpu_device)
    q_out = torch.full((rows, nh, hd), 5.0, dtype=dtype, device=gpu_device) if nh else None
    got = kv.append(d[:, nh:nh + nkv], d[:, nh + nkv:], _int(seq), _int(at), _int(table), rotary=rotary, q=d[:, :nh] if nh else None,
                    q_out=q_out, rotary_pos=_int(turn))
    assert got is q_out
    raw = heads[:, nh:nh + nkv]
    keys = rotate64(raw, turn, rotary.inv_freq, 1.0, rot, layout) if rot else raw.double()
    err = rotate_bound(raw, rot, layout, 1.0, F32, keys) if rot else torch.zeros_like(keys)
    values = heads[:, nh + nkv:].double()
    _check_append(kv, before, [(keys, err), (values, torch.zeros_like(values))], seq, at, table)
    live = [0 <= int(s) < n_seq and 0 <= int(p) // page < width and int(p) >= 0 and 0 <= int(table[s, int(p) // page]) < n_pages
            for s, p in zip(seq, at)]
    if nh:
        here = torch.tensor(live)
        want = rotate64(heads[:, :nh], turn, rotary.inv_freq, 1.0, rot, layout)
        _within(q_out.cpu()[here], want[here], rotate_bound(heads[:, :nh], rot, layout, 1.0, dtype, want)[here])
        assert (q_out.cpu()[~here] == 5).all()
    # what is read back is what is held, rows without a place are zeros
    for out in (F32, dtype):
        k, v = kv.read(_int(seq), _int(at), _int(table), dtype=out)
        for x, pool, sc in ((k, kv.k, kv.k_scale), (v, kv.v, kv.v_scale)):
            held = dense64(pool, sc)
            want = torch.stack([held[int(table[s, int(p) // page]), :, int(p) % page] if ok else torch.zeros(nkv, hd, dtype=torch.float64)
                                for s, p, ok in zip(seq, at, live)])
            _within(x, want, want.abs() * (HALF[out] + 2.0 ** -24) + TINY[out])
            assert (x.cpu()[~torch.tensor(live)] == 0).all()


def test_append_order_does_not_matter_and_the_later_row_stays(gpu_device):
    """Rows of a block anywhere in the call give the same bits as in order; of two rows for one place the later one alone counts."""
    g = torch.Generator().manual_seed(4)
    nkv, hd, page, block, L = 2, 64, 64, 32, 300
    x = torch.randn((L, 2, nkv, hd), generator=g).to(gpu_device)
    table = torch.randperm(12, generator=g).to(torch.int32).view(2, 6)[:, :5].contiguous().to(gpu_device)
    seq, at = torch.arange(L, device=gpu_device).int() % 2, torch.arange(L, device=gpu_device).int() // 2 + 7
    pools = []
    for order in (torch.arange(L), torch.argsort(seq.cpu(), stable=True), torch.randperm(L, generator=g)):
        kv = PagedKV.allocate(12, page, nkv, hd, I8, scale_block=block)
        o = order.to(gpu_device)
        kv.append(x[o, 0], x[o, 1], seq[o], at[o], table)
        pools.append([t.clone() for t in (kv.k, kv.v, kv.k_scale, kv.v_scale)])
    assert all(torch.equal(a, b) for p in pools for a, b in zip(p, pools[0]))
    kv = PagedKV.allocate(12, page, nkv, hd, I8, scale_block=block)
    y = torch.stack([torch.full((nkv, hd), 8.0), torch.full((nkv, hd), 2.0)]).to(gpu_device)
    twice = torch.zeros(2, dtype=torch.int32, device=gpu_device)
    kv.append(y, y, twice, twice + 5, table)
    k, _ = kv.read(twice[:1], twice[:1] + 5, table, dtype=F32)
    assert torch.allclose(kv.k_scale[int(table[0, 0]), :, 0], torch.tensor(2 / 127, device=gpu_device))
    assert float((k - 2).abs().max()) <= 2.0 ** -20


@pytest.mark.parametrize('cache', [I8, E4M3])
def test_append_step_by_step_keeps_what_is_held(gpu_device, cache):
    """One position a call: the scale is the largest so far, a value is off by half a step for each time that it grew."""
    g = torch.Generator().manual_seed(7)
    kv = PagedKV.allocate(4, 32, 2, 64, cache, scale_block=16)
    table = _int([[2, 0]])
    x = torch.randn((40, 2, 64), generator=g) * torch.linspace(0.2, 3, 40)[:, None, None]
    zero = _int([0])
    for p in range(40):
        kv.append(x[p:p + 1].to(gpu_device), -x[p:p + 1].to(gpu_device), zero, _int([p]), table)
    k, v = kv.read(torch.zeros(40, dtype=torch.int32, device=gpu_device), _int(range(40)), table, dtype=F32)
    for b in range(3):
        part = x[16 * b:min(40, 16 * b + 16)].double()
        top = part.abs().amax(-1).cummax(0).values / MOST[cache]                  # [positions, heads]
        sc = kv.k_scale[[2, 2, 0][b], :, b % 2].double().cpu()
        assert float((sc / top[-1] - 1).abs().max()) <= 2.0 ** -21
        for i in range(len(part)):
            steps = sorted(set(float(t) for h in range(2) for t in top[i:, h]))
            half = sum(steps) * 0.5 if cache == I8 else None
            err = (k[16 * b + i].double().cpu() - part[i]).abs()
            if cache == I8:
                assert float(err.max()) <= half * (1 + 2.0 ** -18)
            else:
                n = len(steps)
                assert float((err - part[i].abs() * ((1 + 2.0 ** -4) ** n - 1) - sum(steps) * 2.0 ** -10).max()) <= 1e-9
    assert torch.equal(v, -k)


def test_append_extremes(gpu_device):
    """Zeros, tiny and huge magnitudes, infinities, NaN: within their block and head."""
    for cache in (I8, E4M3):
        kv = PagedKV.allocate(3, 16, 2, 64, cache, scale_block=16)
        x = torch.ones((3, 2, 64), device=gpu_device)
        x[0, 0], x[0, 1] = 0, 2.0 ** -80
        x[1, 0, :4] = torch.tensor([math.inf, -math.inf, 1e30, 1.0])
        x[2, 0, 3] = math.nan
        seq, at, table = _int([0, 0, 0]), _int([0, 16, 32]), _int([[2, 1, 0]])
        kv.append(x, x, seq, at, table)
        for read in kv.read(seq, at, table, dtype=F32):
            assert (read[0] == 0).all()
            top = 2.0 ** 60 * MOST[cache]
            assert read[1, 0, :3].tolist() == [top, -top, top] and abs(float(read[1, 0, 3])) <= 1
            assert float((read[1, 1] - 1).abs().max()) <= 2.0 ** -8
            assert float((read[2, 1] - 1).abs().max()) <= 2.0 ** -8
            if cache == I8:
                assert read[2, 0].isnan().all()
            else:
                assert read[2, 0, 3].isnan() and float((read[2, 0, torch.arange(64) != 3] - 1).abs().max()) <= 2.0 ** -4
        assert (kv.k_scale[2] == 2.0 ** -60).all()
        # an int8 block stays NaN until it begins anew
        kv.append(x[1:2], x[1:2], _int([0]), _int([33]), table)
        assert (cache == I8) == bool(kv.k_scale[0, 0].isnan())
        kv.append(torch.ones_like(x[:1]), torch.ones_like(x[:1]), _int([0]), _int([32]), table)
        assert float((kv.read(_int([0]), _int([32]), table, dtype=F32)[0] - 1).abs().max()) <= 2.0 ** -8


def test_read_other_caches_and_views(gpu_device):
    """16-bit and per-head e4m3 caches are read too, into views, and rows may repeat."""
    g = torch.Generator().manual_seed(9)
    table, seq, at = _int([[1, 0, 2]]), _int([0, 0, 0, -1, 0]), _int([3, 40, 3, 0, 48])
    for cache in (F16, BF16, E4M3):
        sc = [(torch.rand(2, generator=g) + 0.5).to(gpu_device) for _ in range(2)] if cache == E4M3 else [None, None]
        k, v = (torch.randn((3, 2, 16, 64), generator=g).to(cache).to(gpu_device) for _ in range(2))
        kv = PagedKV(k, v, *sc)
        wide = torch.full((2, 5, 3, 72), 9.0, device=gpu_device)
        out = (wide[0, :, :2, :64], wide[1, :, :2, :64])
        got = kv.read(seq, at, table, out=out)
        assert got[0] is out[0] and (wide[:, :, 2] == 9).all() and (wide[..., 64:] == 9).all()
        for x, pool, s in zip(got, (k, v), sc):
            f = pool.float() * (s[:, None, None] if s is not None else 1)
            want = torch.stack([f[1, :, 3], f[2, :, 8], f[1, :, 3], f[0, :, 0] * 0, f[0, :, 0] * 0])
            assert torch.equal(x, want)


# ------------------------------------------------------------------------------------------------ attention
def _batch(g, q_lens, kv_lens, groups, nh, nkv, hd, page, block, dtype, cache, dev, spread=0.0):
    """A batch whose unheld rows are codes of large values, and whose blocks without any held row have NaN scales."""
    q, k, v, table, _ = paged_batch(g, q_lens, kv_lens, groups, nh, nkv, hd, page, dtype, F32, dev, fill=0.0)
    held = torch.zeros(k.shape[:1] + (page,), dtype=torch.bool)
    for s, n in enumerate(kv_lens):
        p = np.arange(n)
        held[table.cpu().numpy()[s][p // page], p % page] = True
    out = []
    for x in (k, v):
        x = x.cpu() * torch.exp2(spread * torch.randn((x.shape[0], nkv, page // block, 1, 1), generator=g)).expand(-1, -1, -1, block, -1).flatten(2, 3)
        codes, scale = coded(x, cache, block)
        c = codes.view(torch.int8)
        c[~held.unsqueeze(1).expand(-1, nkv, -1)] = -128 if cache == I8 else 0x7f
        scale[~held.unflatten(1, (-1, block)).any(-1).unsqueeze(1).expand(-1, nkv, -1)] = math.nan
        out += [codes.to(dev), scale.to(dev)]
    return q, out, table


def _attend(dev, q_lens, kv_lens, groups, nh, nkv, hd, page, block, dtype, cache, seed=0, spread=0.0):
    g = torch.Generator().manual_seed(seed)
    q, (k, ks, v, vs), table = _batch(g, q_lens, kv_lens, groups, nh, nkv, hd, page, block, dtype, cache, dev, spread)
    kv = PagedKV(k, v, ks, vs)
    plan = AttentionPlan(nh, nkv, hd, max_rows=max(1, sum(q_lens)), max_seqs=len(q_lens)).set(q_lens, kv_lens, groups)
    lse = torch.full(q.shape[:2], 3.0, device=dev)
    out = plan.run(q, kv, table, lse=lse)
    torch.cuda.synchronize()
    want, wl, bound = attend_blocks64(q, k, ks, v, vs, table, q_lens, kv_lens, hd ** -0.5)
    # (values past fp16's largest become infinite; within the bound of it either may be)
    big = want.abs() + bound >= torch.finfo(dtype).max
    assert torch.equal(out.isinf().cpu() & ~big, torch.zeros_like(big)) and not out.isnan().any()
    certain = want.abs() - bound >= torch.finfo(dtype).max * (1 + HALF[dtype])
    assert torch.equal(out.double().cpu()[certain], torch.copysign(torch.tensor(math.inf, dtype=torch.float64), want[certain]))
    _within(out, torch.where(big, math.nan, want), bound)
    got = lse.double().cpu()
    assert torch.equal(got == -math.inf, wl == -math.inf)
    seen = wl > -math.inf
    assert float((got - wl)[seen].abs().max() if seen.any() else 0) <= 2.0 ** -15 * (1 + float(wl[seen].abs().max() if seen.any() else 0))
    return plan, q, kv, table, out


TYPES = [(F16, I8), (BF16, I8), (F16, E4M3), (BF16, E4M3)]


@pytest.mark.parametrize('dtype,cache', TYPES)
@pytest.mark.parametrize('hd', [64, 128])
@pytest.mark.parametrize('q_lens,kv_lens,groups,nh,nkv,page,block', [
    ([1], [1], None, 2, 1, 16, 16),
    ([1], [733], None, 14, 2, 16, 16),
    ([1] * 5, [5, 64, 65, 1, 300], None, 4, 4, 48, 16),
    ([1] * 16, [2048 // 8 + i * 9 for i in range(16)], [(16, 256)], 12, 2, 32, 32),
    ([1] * 40, [515 + i for i in range(40)], [(20, 512), (20, 448)], 28, 4, 64, 64),
    ([3, 0, 1, 9], [200, 90, 150, 160], [(4, 80)], 12, 2, 16, 16),
    ([40, 7], [140, 107], [(2, 96)], 28, 4, 32, 16),
    ([2, 5, 1], [0, 3, 0], None, 6, 2, 16, 16),
    ([33, 70], [33, 70], None, 8, 1, 128, 128),
    ([9, 9, 20], [98, 99, 110], [(3, 96)], 32, 1, 96, 48),
])
def test_attention(gpu_device, dtype, cache, hd, q_lens, kv_lens, groups, nh, nkv, page, block):
    print(f'attend blocks {dtype} {cache} {hd} {q_lens} {kv_lens} {groups} {nh} {nkv} {page} {block}', flush=True)
    _attend(gpu_device, q_lens, kv_lens, groups, nh, nkv, hd, page, block, dtype, cache, seed=len(q_lens) + hd)


@pytest.mark.parametrize('dtype,cache', TYPES)
def test_attention_over_scales_far_apart(gpu_device, dtype, cache):
    """Blocks whose values differ by many powers of two: small ones keep their precision in rows that see nothing else."""
    for spread in (3.0, 8.0):
        _attend(gpu_device, [1] * 6, [40, 16, 300, 17, 200, 90], None, 4, 2, 64, 32, 16, dtype, cache, seed=3, spread=spread)
        _attend(gpu_device, [60, 33], [200, 33], None, 4, 2, 128, 32, 16, dtype, cache, seed=4, spread=spread)


@pytest.mark.parametrize('seed', range(16))
def test_random_batches(gpu_device, seed):
    rng = np.random.default_rng(2000 + seed)
    nkv = int(rng.choice([1, 2, 3, 4]))
    nh = nkv * int(rng.choice([1, 2, 5, 6, 7, 16, 32]))
    hd = int(rng.choice([64, 128]))
    page, block = [(16, 16), (32, 16), (48, 48), (64, 32), (128, 64), (96, 32)][int(rng.integers(6))]
    dtype, cache = TYPES[seed % 4]
    q_lens, kv_lens, groups = [], [], []
    for _ in range(rng.integers(1, 4)):
        size, shared = int(rng.integers(1, 7)), int(rng.integers(0, 700)) // page * page
        for _ in range(size):
            q_lens.append(int(rng.choice([0, 1, 1, 1, 2, 5, 9, 33, 70])))
            kv_lens.append(shared + int(rng.integers(0, 260)))
        groups.append((size, shared))
    print(f'random blocks {seed}: {nh}/{nkv} heads of {hd}, {page} {block}, {dtype} {cache}, {q_lens} {kv_lens} {groups}', flush=True)
    _attend(gpu_device, q_lens, kv_lens, groups, nh, nkv, hd, page, block, dtype, cache, seed=seed)


def test_long_contexts(gpu_device):
    _attend(gpu_device, [1], [20000], None, 2, 1, 64, 16, 16, F16, I8, seed=1)
    _attend(gpu_device, [1, 1, 1], [9003, 9100, 9001], [(3, 8992)], 28, 4, 128, 32, 16, BF16, I8, seed=2)
    _attend(gpu_device, [130], [3000], None, 4, 4, 64, 128, 64, F16, E4M3, seed=4)


@pytest.mark.parametrize('dtype,cache', TYPES)
def test_hidden_pages_and_poisoned_blocks(gpu_device, dtype, cache):
    """Entries outside the pool hide their positions; a NaN scale or e4m3 NaN reaches the rows that see its position and no others;
    pages that were only cleared count as zeros."""
    g = torch.Generator().manual_seed(11)
    q_lens, kv_lens = [1, 20, 2, 1], [300, 290, 20, 16]
    q, (k, ks, v, vs), table = _batch(g, q_lens, kv_lens, None, 14, 2, 128, 16, 16, dtype, cache, gpu_device)
    table[0, 5], table[0, 17], table[1, 18], table[2] = k.shape[0], -1, -(1 << 31), -7
    kv = PagedKV(k, v, ks, vs)
    plan = AttentionPlan(14, 2, 128, max_rows=24, max_seqs=4).set(q_lens, kv_lens)
    lse = torch.zeros(24, 14, device=gpu_device)
    out = plan.run(q, kv, table, lse=lse)
    want, wl, bound = attend_blocks64(q, k, ks, v, vs, table, q_lens, kv_lens, 128 ** -0.5)
    _within(out, want, bound)
    assert torch.equal(lse.cpu() == -math.inf, wl == -math.inf) and (out[21:23] == 0).all()
    # position 271 (of rows 1.. of sequence 1, whose first query stands at 270) becomes NaN
    e = int(table[1, 271 // 16])
    if cache == I8:
        vs[e, 0, 0] = math.nan
        first = 256                                            # the whole block
    else:
        v.view(torch.uint8)[e, 0, 271 % 16, 5] = 0x7f
        first = 271
    out2 = plan.run(q, kv, table)
    bad = torch.zeros(24, 14, 128, dtype=torch.bool)
    for i in range(20):
        if 270 + i >= first:
            bad[1 + i, :7, slice(None) if cache == I8 else 5] = True
    assert torch.equal(out2.isnan().cpu(), bad)
    assert torch.equal(out2.cpu()[~bad], out.cpu()[~bad])
    fresh = PagedKV.allocate(4, 16, 2, 128, cache, scale_block=16)
    t = _int([[0, 1, 2]])
    one = AttentionPlan(14, 2, 128, max_rows=1, max_seqs=1).set([1], [40])
    lse = torch.zeros(1, 14, device=gpu_device)
    assert (one.run(q[:1], fresh, t, lse=lse) == 0).all()
    assert float((lse - math.log(40)).abs().max()) <= 2.0 ** -15 * 5


def test_pools_past_32_bits(gpu_device):
    """Pages, codes and scales behind 2^32 bytes of a pool: append, read, attention and the page pool's copies."""
    from seedplane_amd.pages import PagePool
    g = torch.Generator().manual_seed(13)
    nkv, page, hd, n = 2, 128, 128, 140000                    # 4.6 GB of keys, as much of values
    pools = [torch.empty((n, nkv, page, hd), dtype=I8, device=gpu_device) for _ in range(2)]
    scales = [torch.ones((n, nkv, page // 16), device=gpu_device) for _ in range(2)]
    kv = PagedKV(*pools, *scales)
    table = _int([[n - 1, 3, n - 2], [7, n - 3, 5]])
    seq, at = _int([0] * 300 + [1] * 270), _int(list(range(300)) + list(range(270)))
    x = torch.randn((570, 6, hd), generator=g).half().to(gpu_device)
    q = kv.append(x[:, 2:4], x[:, 4:], seq, at, table, rotary=Rotary(hd, theta=1e6), q=x[:, :2])
    lens = [300, 270]
    plan = AttentionPlan(2, nkv, hd, 2, 2).set([1, 1], lens)
    out = plan.run(q[[299, 569]].contiguous(), kv, table)
    used = torch.unique(table.view(-1)).long()
    small = torch.zeros_like(table)
    for i, e in enumerate(used.tolist()):
        small[table == e] = i
    args = [t[used] for p in zip(pools, scales) for t in p]
    want, _, bound = attend_blocks64(q[[299, 569]], *args, small, [1, 1], lens, hd ** -0.5)
    _within(out, want, bound)
    k, v = kv.read(seq, at, table, dtype=F32)
    held = dense64(args[2], args[3])
    pos = at.cpu().long()
    _within(v, torch.stack([held[int(small[s, p // page]), :, p % page] for s, p in zip(seq.tolist(), pos.tolist())]), torch.full((570, nkv, hd), 1e-6, dtype=torch.float64))
    pool = PagePool(kv, 2, 3)
    pool.copy(_int([n - 1, 3]), _int([11, n - 9]))
    for p in (pools[0], pools[1], scales[0], scales[1]):
        assert torch.equal(p[11], p[n - 1]) and torch.equal(p[n - 9], p[3])


def test_serving_run_captured(gpu_device):
    """A prompt appended, then steps of append and attention in a graph that follows positions on the device; every step against the
    64-bit form over what the cache holds, and against the eager calls in every bit."""
    g = torch.Generator().manual_seed(21)
    nh, nkv, hd, page, B = 12, 2, 128, 32, 3
    rotary = Rotary(hd, theta=1e6)
    start = [37, 5, 64]
    table = torch.randperm(B * 4, generator=g).int().view(B, 4).to(gpu_device)
    eager, graph = (PagedKV.allocate(B * 4, page, nkv, hd, I8, scale_block=16) for _ in range(2))
    seq = _int(np.repeat(range(B), start))
    pos = _int(np.concatenate([np.arange(n) for n in start]))
    x = torch.randn((sum(start), nh + 2 * nkv, hd), generator=g).half().to(gpu_device)
    for kv in (eager, graph):
        kv.append(x[:, nh:nh + nkv], x[:, nh + nkv:], seq, pos, table, rotary=rotary, q=x[:, :nh])
    plans = [AttentionPlan(nh, nkv, hd, B, B) for _ in range(2)]
    step = torch.zeros((B, nh + 2 * nkv, hd), dtype=F16, device=gpu_device)
    each, at = _int(range(B)), _int(start)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    plans[1].set([1] * B, [n + 1 for n in start])
    tape = torch.cuda.CUDAGraph()
    with torch.cuda.graph(tape, stream=side):
        qr = graph.append(step[:, nh:nh + nkv], step[:, nh + nkv:], each, at, table, rotary=rotary, q=step[:, :nh])
        out = plans[1].run(qr, graph, table)
    for i in range(20):
        step.copy_(torch.randn(step.shape, generator=g).half())
        at.copy_(torch.tensor([n + i for n in start], dtype=torch.int32))
        lens = [n + i + 1 for n in start]
        for p in plans:
            p.set([1] * B, lens)
        tape.replay()
        q = eager.append(step[:, nh:nh + nkv], step[:, nh + nkv:], each, at, table, rotary=rotary, q=step[:, :nh])
        want = plans[0].run(q, eager, table)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(graph.k, eager.k) and torch.equal(graph.v_scale, eager.v_scale)
        ref, _, bound = attend_blocks64(q, eager.k, eager.k_scale, eager.v, eager.v_scale, table, [1] * B, lens, hd ** -0.5)
        _within(want, ref, bound)
