"""Long calls over paged caches with a scale per block.  Appends of many rows: workgroups that take several blocks and look their rows up at once, or,
where too many rows are near, block by block.  Attention: items of more positions than their tables hold.  Tolerances: tests/blocks_ref.py."""
import pytest
import torch

from blocks_ref import attend_blocks64
from paged_ref import rotate64, rotate_bound
from seedplane_amd.paged import AttentionPlan, PagedKV, Rotary
from test_gpu_blocks import BF16, E4M3, F16, F32, I8, _cache, _check_append, _int, _within

pytestmark = pytest.mark.gpu


def _spots(g, rows, n_seq, far, order):
    """Sequences and positions of a call's rows: 'runs': one sequence after the other; 'time': a position of every sequence after the
    other; 'any': all mixed."""
    spots = torch.randperm(n_seq * far, generator=g)[:rows]
    seq, at = spots // far, spots % far
    if order == 'any':
        return seq.int(), at.int()
    by = (seq * far + at if order == 'runs' else at * n_seq + seq).argsort()
    return seq[by].int(), at[by].int()


@pytest.mark.parametrize('cache', [I8, E4M3])
@pytest.mark.parametrize('rows,nh,nkv,hd,rot,page,block,layout,order,n_seq,far,dtype', [
    (4097, 3, 2, 32, 32, 32, 16, 'half', 'runs', 3, 1500, F16), (4099, 0, 1, 32, 0, 64, 64, 'half', 'time', 40, 110, BF16),
    (4102, 1, 1, 40, 24, 48, 48, 'interleaved', 'any', 5, 900, F32), (9001, 0, 3, 16, 16, 16, 16, 'half', 'runs', 1, 9100, BF16),
    (4500, 2, 2, 12, 12, 32, 16, 'half', 'time', 3, 1600, F16), (4401, 0, 1, 128, 128, 128, 128, 'half', 'runs', 4, 1200, BF16),
    (300, 1, 1, 128, 128, 256, 128, 'interleaved', 'any', 2, 300, F16), (8200, 0, 1, 32, 32, 16, 16, 'half', 'runs', 700, 12, F16)])
def test_long_append(gpu_device, cache, rows, nh, nkv, hd, rot, page, block, layout, order, n_seq, far, dtype):
    print(f'long append {cache} {rows} {nh} {nkv} {hd} {rot} {page} {block} {layout} {order} {n_seq} {dtype}', flush=True)
    g = torch.Generator().manual_seed(rows + hd)
    width = -(-far // page)
    n_pages = n_seq * width + 2
    table = torch.randperm(n_pages, generator=g)[:n_seq * width].to(torch.int32).view(n_seq, width)
    seq, at = _spots(g, rows, n_seq, far, order)
    seq[::11] = -1                                             # a padded batch
    seq[7], at[9], at[13] = n_seq, -5, width * page
    table[int(seq[1]), int(at[1]) // page] = n_pages
    kv = _cache(g, gpu_device, n_pages, nkv, page, hd, cache, block)
    before = [(kv.k.clone(), kv.k_scale.clone()), (kv.v.clone(), kv.v_scale.clone())]
    heads = (torch.randn((rows, nh + 2 * nkv, hd), generator=g) * torch.rand((rows, 1, 1), generator=g) * 2).to(dtype)
    turn = torch.randint(0, 100000, (rows,), generator=g).to(torch.int32)
    rotary = Rotary(hd, theta=1e6, rot_dim=rot, layout=layout) if rot else None
    d = heads.to(gpu_device)
    q_out = torch.empty((rows, nh, hd), dtype=dtype, device=gpu_device) if nh else None
    kv.append(d[:, nh:nh + nkv], d[:, nh + nkv:], _int(seq), _int(at), _int(table), rotary=rotary, q=d[:, :nh] if nh else None, q_out=q_out,
              rotary_pos=_int(turn))
    raw = heads[:, nh:nh + nkv]
    keys = rotate64(raw, turn, rotary.inv_freq, 1.0, rot, layout) if rot else raw.double()
    err = rotate_bound(raw, rot, layout, 1.0, F32, keys) if rot else torch.zeros_like(keys)
    values = heads[:, nh + nkv:].double()
    _check_append(kv, before, [(keys, err), (values, torch.zeros_like(values))], seq, at, table)


@pytest.mark.parametrize('n_seq,far', [(1, 6000), (5, 1100), (300, 20)])
def test_long_append_order_does_not_matter(gpu_device, n_seq, far):
    """The same rows in three orders, and in calls of fewer rows that split no block: the same codes and scales."""
    g = torch.Generator().manual_seed(n_seq)
    nkv, hd, page, block, rows = 2, 64, 32, 16, 5003
    width = -(-far // page)
    table = torch.randperm(n_seq * width, generator=g).to(torch.int32).view(n_seq, width)
    seq, at = _spots(g, rows, n_seq, far, 'runs')
    x = torch.randn((2, rows, nkv, hd), generator=g).to(BF16)
    rotary = Rotary(hd)
    start = _cache(g, gpu_device, n_seq * width, nkv, page, hd, I8, block)
    pools = (start.k, start.v, start.k_scale, start.v_scale)

    def of(calls):
        kv = PagedKV(*(p.clone() for p in pools))
        for rows_of in calls:
            k, v = (t[rows_of].to(gpu_device) for t in x)
            kv.append(k, v, _int(seq[rows_of]), _int(at[rows_of]), _int(table), rotary=rotary)
        return kv
    blocks = seq.long() * (far // block + 1) + at // block
    want = of([(blocks % 3 == i).nonzero()[:, 0] for i in range(3)])
    for order in (torch.arange(rows), (at.long() * n_seq + seq).argsort(), torch.randperm(rows, generator=g)):
        got = of([order])
        for a, b in zip((want.k, want.v, want.k_scale, want.v_scale), (got.k, got.v, got.k_scale, got.v_scale)):
            assert torch.equal(a, b)


@pytest.mark.parametrize('cache', [I8, E4M3])
@pytest.mark.parametrize('q_len,n_seq,hd,dtype', [(4, 600, 128, F16), (8, 600, 128, BF16), (8, 560, 64, F16), (3, 600, 64, BF16), (1, 1100, 128, BF16)])
def test_items_longer_than_their_table(gpu_device, q_len, n_seq, hd, dtype, cache):
    """So many sequences that none is cut: each item brings the rows of its positions to LDS several times, of tiles of 32, 64 and
    128 rows.  All sequences name the same pages, in orders of their own, and a few of them are compared."""
    print(f'long items {q_len} {n_seq} {hd} {dtype} {cache}', flush=True)
    g = torch.Generator().manual_seed(q_len + hd)
    nh, page, n = 16, 64, 4500
    width = -(-n // page)
    kv = _cache(g, gpu_device, width, 1, page, hd, cache, 16)
    table = torch.stack([torch.randperm(width, generator=g) for _ in range(n_seq)]).int()
    lens = [n - int(i) for i in torch.randint(0, 60, (n_seq,), generator=g)]
    q = torch.randn((n_seq * q_len, nh, hd), generator=g).to(dtype).to(gpu_device)
    plan = AttentionPlan(nh, 1, hd, max_rows=n_seq * q_len, max_seqs=n_seq).set([q_len] * n_seq, lens)
    out = plan.run(q, kv, table.to(gpu_device))
    for s in (0, n_seq // 2, n_seq - 1):
        rows = slice(s * q_len, (s + 1) * q_len)
        want, _, bound = attend_blocks64(q[rows], kv.k, kv.k_scale, kv.v, kv.v_scale, table[s:s + 1], [q_len], [lens[s]], hd ** -0.5)
        _within(out[rows], want, bound)
