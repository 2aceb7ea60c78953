"""Calls at the edges of the page pool and of beam search's selection."""
import numpy as np
import pytest
import torch

from seedplane_amd.beam import beam_select
from seedplane_amd.paged import PagedKV
from seedplane_amd.pages import PagePool
from test_gpu_beam import _check
from test_gpu_pages import Both, F16, I8, _caches, _int

pytestmark = pytest.mark.gpu


def test_lengths_outside_the_table_stay_in_it(gpu_device):
    """A program may set the tables; a length below 0 counts as 0, one past the table's width as the width."""
    g = torch.Generator().manual_seed(0)
    pool = PagePool(_caches(g, 1, 12, 1, 16, 16, F16), 3, 3)
    guard = pool.table.clone()
    pool.lengths.copy_(_int([-(1 << 31), 1 << 30, -17]))
    pool.grow(_int([20, 0, 0]))
    assert pool.lengths.tolist() == [20, 48, 0]
    guard[0, :2] = _int([0, 1])
    assert torch.equal(pool.table, guard) and pool.holders.tolist() == [1, 1] + [0] * 10 and pool.missing.tolist() == [0]
    pool.lengths[2] = -5
    pool.fork(_int([2, 0, 1]))
    assert pool.lengths.tolist() == [0, 20, 48] and pool.table[1].tolist() == [0, 1, -1] and pool.table[0].tolist() == [-1] * 3


def test_counts_past_every_width(gpu_device):
    """The largest counts fill the table's width and are counted."""
    g = torch.Generator().manual_seed(1)
    pool = PagePool(_caches(g, 1, 8, 1, 16, 16, I8, 16), 3, 4)
    pool.grow(_int([2 ** 31 - 1, -2 ** 31, 5]))
    assert pool.lengths.tolist() == [64, 0, 5] and pool.missing.tolist() == [1]
    assert pool.table.tolist() == [[0, 1, 2, 3], [-1] * 4, [4, -1, -1, -1]]


@pytest.mark.parametrize('page,nkv,hd', [(1, 1, 2), (1, 3, 16), (5, 2, 6), (128, 1, 64)])
def test_lives_on_other_pages(gpu_device, page, nkv, hd):
    """Pages of one position (no last page is ever shared), odd ones, large ones."""
    g = torch.Generator().manual_seed(page)
    rng = np.random.default_rng(page)
    both = Both(_caches(g, 2, 40, nkv, page, hd, F16), 5, 9)
    for _ in range(12):
        both.do('grow', rng.integers(0, 2 * page + 1, 5).tolist())
        both.do('fork', rng.integers(-1, 5, 5).tolist())
        both.do('compact')
        both.do('free', [int(rng.integers(0, 5))])


@pytest.mark.parametrize('hd,dtype,first', [(6, I8, 0), (36, I8, 0), (40, I8, 0), (7, F16, 0), (32, F16, 1), (32, I8, 4)])
def test_copies_of_rows_of_any_width(gpu_device, hd, dtype, first):
    """Rows of bytes, of 4 bytes, and pools that begin `first` values behind an aligned address."""
    g = torch.Generator().manual_seed(hd)
    caches = []
    for _ in range(2):
        base = [torch.randint(0, 100, (first + 20 * 2 * 16 * hd,), generator=g, dtype=torch.int8).to(gpu_device).to(dtype) for _ in range(2)]
        pools = [b[first:].view(20, 2, 16, hd) for b in base]
        scales = [torch.rand((20, 2, 1), generator=g).to(gpu_device) for _ in range(2)] if dtype == I8 else [None, None]
        caches.append(PagedKV(*pools, *scales))
    both = Both(caches, 4, 5)
    both.do('grow', [21, 3, 0, 33])
    both.do('fork', [0, 0, 3, 0])
    both.do('free', [1])
    both.do('compact')


def test_steps_into_the_scores_that_they_read(gpu_device):
    """A step's buffers taken for the next one: its scores are read before they are written."""
    g = torch.Generator().manual_seed(2)
    x = [(4 * torch.randn((15, 700), generator=g)).to(gpu_device) for _ in range(4)]
    scores = torch.zeros((3, 5), device=gpu_device)
    want, step = scores, None
    for logits in x:
        apart = beam_select(logits, want, eos=3)
        want = apart.next_scores
        step = beam_select(logits, scores if step is None else step.next_scores, eos=3, out=step)
        for a, b in zip(apart, step):
            assert torch.equal(a, b)


def test_selections_side_by_side(gpu_device):
    """Two streams at once: each call has a workspace of its own."""
    g = torch.Generator().manual_seed(3)
    x = [torch.randn((24, 30000), generator=g).to(gpu_device) for _ in range(2)]
    scores = torch.zeros((3, 8), device=gpu_device)
    want = [beam_select(t, scores) for t in x]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(beam_select(x[i], scores))
    torch.cuda.synchronize()
    for i in range(2):
        for step in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(step, want[i]))


def test_ends_that_are_no_tokens_are_refused(gpu_device):
    x, s = torch.zeros((2, 9), device=gpu_device), torch.zeros((1, 2), device=gpu_device)
    for eos in (-1, 1 << 31, 1 << 40, [3, -2]):
        with pytest.raises(ValueError):
            beam_select(x, s, eos=eos)
    assert beam_select(x, s, eos=(1 << 31) - 1).next_tokens.tolist() == [[0, 1]]


@pytest.mark.parametrize('dtype', [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize('B,K,n,V', [(1, 4, 8, 40000), (2, 3, 64, 33001), (5, 8, 16, 9000), (1, 1, 1, 20000), (1, 16, 33, 5000)])
@pytest.mark.parametrize('kind', ['equal', 'lowest', 'padded', 'falling', 'rising', 'one thread', 'few values', 'zeros', 'one beam', 'few'])
def test_where_the_best_lie(gpu_device, kind, B, K, n, V, dtype):
    """Rows in which more values than the buffers hold are as good as the n-th best, or the best lie side by side, at strides, at the end,
    in one beam."""
    print(f'selection {kind} {B} {K} {n} {V} {dtype}', flush=True)
    g = torch.Generator().manual_seed(V + n)
    x = torch.randn((B * K, V), generator=g)
    at = torch.arange(V)
    low = torch.finfo(dtype).min
    scores = -torch.arange(K, dtype=torch.float32).repeat(B, 1) * 0.37
    if kind == 'equal':
        x.fill_(1.5)
    elif kind == 'lowest':                                     # a mask of the type's lowest value, a few tokens allowed
        x = torch.where(torch.rand((B * K, V), generator=g) < 30 / V, x, low)
    elif kind == 'padded':
        x[:, V // 3:] = -10000.0
    elif kind == 'falling':
        x = x.sort(1, descending=True).values
    elif kind == 'rising':
        x = x.sort(1).values
    elif kind == 'one thread':                                 # 8 of every 2048 values
        x = x + 10.0 * (at % 2048 < 8)
    elif kind == 'few values':
        x = torch.randint(0, 3, (B * K, V), generator=g).float()
    elif kind == 'zeros':                                      # of both signs: equal
        x = torch.where(torch.rand((B * K, V), generator=g) < 0.5, -0.0, 0.0)
    elif kind == 'one beam':
        scores = scores * 100
    else:
        x = torch.where(torch.rand((B * K, V), generator=g) < n / 2 / V, x, -torch.inf)
    _check(x.to(dtype).to(gpu_device), scores.to(gpu_device), n=n)
