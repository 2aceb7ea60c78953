"""The page pool on the GPU against its rules on lists: tables, holders, what is copied in every layer and what is left alone."""
import numpy as np
import pytest
import torch

from pages_ref import Pages
from seedplane_amd.paged import PagedKV
from seedplane_amd.pages import PagePool

pytestmark = pytest.mark.gpu

F16, I8, E4M3 = torch.float16, torch.int8, torch.float8_e4m3fn


def _int(x):
    return torch.as_tensor(x, dtype=torch.int32, device='cuda')


def _caches(g, layers, n_pages, nkv, page, hd, dtype, block=None, layout='heads'):
    caches = []
    for _ in range(layers):
        if layout == 'heads':
            shape = (n_pages, nkv, page, hd)
            view = lambda t: t
        elif layout == 'rows':                               # [pages, rows, heads, values]
            shape = (n_pages, page, nkv, hd)
            view = lambda t: t.transpose(1, 2)
        else:                                                # wider rows, pages and heads apart
            shape = (n_pages, nkv + 1, page + 1, hd + 16)
            view = lambda t: t[:, :nkv, :page, :hd]
        pools = [view(torch.randint(0, 100, shape, generator=g, dtype=torch.int8).cuda().to(dtype) if dtype != E4M3 else
                      torch.randint(0, 100, shape, generator=g, dtype=torch.int8).cuda().view(E4M3)) for _ in range(2)]
        scales = [torch.rand((n_pages, nkv, page // block), generator=g).cuda() for _ in range(2)] if block else [None, None]
        caches.append(PagedKV(*pools, *scales))
    return caches


def _bytes(t):
    return t.contiguous().view(torch.uint8).cpu() if t.element_size() == 1 else t.cpu()


class Both:
    """A pool and its rules, changed together and compared."""

    def __init__(self, caches, max_seqs, width):
        self.pool = PagePool(caches, max_seqs, width)
        kv = caches[0]
        self.ref = Pages(kv.n_pages, kv.page_size, max_seqs, width)

    def held(self):
        return [_bytes(t) for c in self.pool.caches for t in (c.k, c.v)], \
            [s.cpu() for c in self.pool.caches for s in (c.k_scale, c.v_scale) if s is not None]

    def do(self, name, arg=None):
        pools, scales = self.held()
        got = getattr(self.pool, name)(*(() if arg is None else (_int(arg),)))
        assert got is self.pool
        getattr(self.ref, name)(*(() if arg is None else (arg,)))
        for src, dst, rows in self.ref.copies:
            for p in pools:
                p[dst, :, :rows] = p[src, :, :rows]
            for s in scales:
                n = -(-rows // (self.ref.page // s.shape[2]))
                s[dst, :, :n] = s[src, :, :n]
        self.ref.copies = []
        self.check(pools, scales)

    def check(self, pools, scales):
        assert self.pool.table.tolist() == self.ref.table()
        assert self.pool.lengths.tolist() == self.ref.lengths
        assert self.pool.holders.tolist() == self.ref.holders
        assert self.pool.missing.tolist() == [self.ref.missing]
        for a, b in zip(self.held(), (pools, scales)):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize('dtype,block,layout', [(F16, None, 'heads'), (I8, 16, 'heads'), (E4M3, 16, 'rows'), (F16, None, 'apart'), (I8, 32, 'apart')])
@pytest.mark.parametrize('seed', range(3))
def test_random_lives_of_sequences(gpu_device, dtype, block, layout, seed):
    """Growth, forks, ends and compaction in random order, the pool running short of pages now and then."""
    rng = np.random.default_rng(100 * seed + 7)
    S, width, page, layers = int(rng.integers(1, 40)), int(rng.integers(2, 9)), 32, int(rng.integers(1, 4))
    nkv, hd = int(rng.integers(1, 4)), int(rng.choice([16, 64, 24]))
    n_pages = max(4, S * width // 2)
    print(f'pages {dtype} {block} {layout}: {S} sequences of {width}, {n_pages} pages, {layers} layers, {nkv} heads of {hd}', flush=True)
    both = Both(_caches(torch.Generator().manual_seed(seed), layers, n_pages, nkv, page, hd, dtype, block, layout), S, width)
    for i in range(25):
        what = rng.choice(['grow', 'grow', 'fork', 'free', 'compact'])
        if what == 'grow':
            both.do('grow', (rng.integers(-3, 50, S) * (rng.random(S) < 0.4)).tolist())
        elif what == 'fork':
            stay = np.arange(S)
            other = rng.integers(-1, S + 1, S)
            both.do('fork', np.where(rng.random(S) < 0.5, stay, other).tolist())
        elif what == 'free':
            both.do('free', rng.integers(-1, S + 2, int(rng.integers(1, S + 1))).tolist())
        else:
            both.do('compact')


def test_many_sequences_and_pages(gpu_device):
    """More sequences than a block has threads, more pages than a scan takes at once, pages near the end."""
    g = torch.Generator().manual_seed(1)
    rng = np.random.default_rng(1)
    both = Both(_caches(g, 1, 30000, 1, 16, 16, I8, 16), 1500, 20)
    both.do('grow', rng.integers(1, 320, 1500).tolist())
    both.do('free', rng.permutation(1500)[:700].tolist())
    both.do('compact')
    both.do('fork', rng.integers(0, 1500, 1500).tolist())
    both.do('grow', [9] * 1500)
    both.do('compact')


def test_kept_pages_and_places(gpu_device):
    """A page that the caller keeps is not given away, moves in a compaction, and its new place is told."""
    g = torch.Generator().manual_seed(2)
    both = Both(_caches(g, 2, 12, 2, 16, 16, F16), 4, 4)
    both.do('grow', [40, 20, 0, 17])
    keep = both.pool.table[3, 0].clone()
    both.pool.holders[keep.long()] += 1
    both.ref.holders[int(keep)] += 1
    both.do('free', [1, 3, 1, 9, -2])
    both.do('grow', [0, 0, 16, 0])
    assert int(both.pool.table[2, 0]) != int(keep)
    both.do('free', [0])
    places = torch.full((12,), 77, dtype=torch.int32, device=gpu_device)
    before = both.pool.caches[1].v[int(keep)].clone()
    both.pool.compact(places)
    assert places.tolist() == both.ref.compact()
    assert torch.equal(both.pool.caches[1].v[int(places[int(keep)])], before)
    assert both.pool.holders.tolist() == both.ref.holders and both.pool.table.tolist() == both.ref.table()


def test_copy(gpu_device):
    g = torch.Generator().manual_seed(3)
    for layout in ('heads', 'rows', 'apart'):
        caches = _caches(g, 3, 9, 2, 32, 24, I8, 16, layout)
        pool = PagePool(caches, 1, 1)
        before = [(c.k.clone(), c.v.clone(), c.k_scale.clone(), c.v_scale.clone()) for c in caches]
        pool.copy(_int([0, 5, 9, -1, 2, 3]), _int([1, 6, 2, 3, 40, 3]))
        for c, b in zip(caches, before):
            for now, was in zip((c.k, c.v, c.k_scale, c.v_scale), b):
                was[1], was[6] = was[0].clone(), was[5].clone()
                assert torch.equal(now, was)
        pool.copy(_int([]), _int([]))


def test_captured(gpu_device):
    """One graph of fork, end, compaction and growth, replayed with other parents each time."""
    g = torch.Generator().manual_seed(4)
    rng = np.random.default_rng(4)
    S, width = 12, 6
    both = Both(_caches(g, 2, 80, 2, 16, 64, F16), S, width)
    both.do('grow', rng.integers(1, 60, S).tolist())
    parents, ends, counts = _int(range(S)), _int([-1, -1]), _int([0] * S)
    tape = torch.cuda.CUDAGraph()
    with torch.cuda.graph(tape):
        both.pool.fork(parents)
        both.pool.free(ends)
        both.pool.compact()
        both.pool.grow(counts)
    for i in range(5):
        pools, scales = both.held()
        p, e, c = rng.integers(0, S, S).tolist(), rng.integers(0, S, 2).tolist(), rng.integers(0, 9, S).tolist()
        parents.copy_(_int(p))
        ends.copy_(_int(e))
        counts.copy_(_int(c))
        tape.replay()
        torch.cuda.synchronize()
        both.ref.fork(p)
        both.ref.free(e)
        both.ref.compact()
        both.ref.grow(c)
        for src, dst, rows in both.ref.copies:
            for t in pools:
                t[dst, :, :rows] = t[src, :, :rows]
        both.ref.copies = []
        both.check(pools, scales)
        torch.zeros(1000, device=gpu_device).add_(1)          # (other work between replays)


def test_refusals(gpu_device):
    g = torch.Generator().manual_seed(5)
    a, b = _caches(g, 2, 8, 2, 16, 64, F16)
    c, = _caches(g, 1, 8, 2, 16, 64, I8, 16)
    other, = _caches(g, 1, 9, 2, 16, 64, F16)
    for caches in ([], [a, c], [a, other]):
        with pytest.raises(ValueError):
            PagePool(caches, 4, 4)
    for sizes in ((0, 4), (4, 0), (65536, 1), (60000, 60000)):
        with pytest.raises(ValueError):
            PagePool([a, b], *sizes)
    pool = PagePool([a, b], 4, 4)
    for call in (lambda: pool.fork(_int([0, 1, 2])), lambda: pool.fork(_int([0, 1, 2, 3]).long()), lambda: pool.grow(torch.zeros(4, dtype=torch.int32)),
                 lambda: pool.free(_int([[0]])), lambda: pool.compact(_int([0] * 7)), lambda: pool.copy(_int([0, 1]), _int([0])),
                 lambda: pool.copy(_int([0, 1, 2, 3])[::2], _int([0, 1]))):
        with pytest.raises(ValueError):
            call()
