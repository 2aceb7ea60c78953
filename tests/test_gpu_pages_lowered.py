"""Sequences whose lengths a program has lowered (drafted positions that were rejected): the pages that their rows still name behind are given back
where growth comes to them, and by forks and ends; none is lost, and none is given to two places."""
import numpy as np
import pytest
import torch

from seedplane_amd.paged import PagedKV
from seedplane_amd.pages import PagePool

pytestmark = pytest.mark.gpu

PAGE = 16


def _int(x):
    return torch.as_tensor(x, dtype=torch.int32, device='cuda')


def _grow(table, lengths, holders, counts, width):
    """The rule on lists; returns the pages that were wanted and not found, and sequences that were cut."""
    missing, places = 0, []
    for s, c in enumerate(counts):
        n = lengths[s] + max(c, 0)
        missing += n > width * PAGE
        n = min(n, width * PAGE)
        places += [(s, j) for j in range(-(-lengths[s] // PAGE), -(-n // PAGE))]
        lengths[s] = n
    for s, j in places:
        if table[s][j] >= 0:
            holders[table[s][j]] -= 1
    free = [e for e, h in enumerate(holders) if h == 0]
    for (s, j), e in zip(places, free + [-1] * len(places)):
        table[s][j] = e
        if e >= 0:
            holders[e] = 1
    return missing + max(0, len(places) - len(free))


@pytest.mark.parametrize('S,width,n_pages', [(1, 4, 4), (5, 7, 20), (40, 9, 200), (300, 12, 2500), (1100, 5, 6000)])
def test_growth_behind_lowered_lengths(gpu_device, S, width, n_pages):
    rng = np.random.default_rng(S)
    pool = PagePool([PagedKV.allocate(n_pages, PAGE, 1, 16)], S, width)
    table, lengths, holders, missing = [[-1] * width for _ in range(S)], [0] * S, [0] * n_pages, 0
    for i in range(12):
        counts = (rng.integers(-3, 60, S) * (rng.random(S) < 0.7)).tolist()
        pool.grow(_int(counts))
        missing += _grow(table, lengths, holders, counts, width)
        assert pool.table.tolist() == table and pool.lengths.tolist() == lengths
        assert pool.holders.tolist() == holders and pool.missing.tolist() == [missing]
        assert sum(holders) == sum(e >= 0 for row in table for e in row) and max(holders) <= 1
        lengths = [int(n * f) if f < 1 else n for n, f in zip(lengths, rng.uniform(0.3, 1.4, S))]
        pool.lengths.copy_(_int(lengths))


def test_drafts_that_are_rejected_lose_no_page(gpu_device):
    """Four positions more each step, all but one taken back: a pool with just the pages that this needs never runs out, and ends empty."""
    S, width = 6, 8
    pool = PagePool([PagedKV.allocate(S * width, PAGE, 1, 16)], S, width)
    for n in range(1, width * PAGE - 3):
        pool.grow(_int([4] * S))
        pool.lengths.sub_(3)
        assert pool.lengths.tolist() == [n] * S and int(pool.missing) == 0
    pool.fork(_int([0, 0, 1, 2, 3, 4]))
    assert int(pool.missing) == 0 and int((pool.holders > 0).sum()) <= S * width
    pool.free(_int(range(S)))
    assert pool.holders.tolist() == [0] * (S * width) and pool.table.tolist() == [[-1] * width] * S


def test_captured(gpu_device):
    S, width, n_pages = 5, 6, 30
    pool = PagePool([PagedKV.allocate(n_pages, PAGE, 1, 16)], S, width)
    counts, tape = _int([0] * S), torch.cuda.CUDAGraph()
    table, lengths, holders, missing = [[-1] * width for _ in range(S)], [0] * S, [0] * n_pages, 0
    with torch.cuda.graph(tape):
        pool.grow(counts)
    rng = np.random.default_rng(9)
    for i in range(6):
        c = rng.integers(0, 40, S).tolist()
        counts.copy_(_int(c))
        tape.replay()
        missing += _grow(table, lengths, holders, c, width)
        assert pool.table.tolist() == table and pool.holders.tolist() == holders and pool.missing.tolist() == [missing]
        lengths = [n // 2 for n in lengths]
        pool.lengths.copy_(_int(lengths))
