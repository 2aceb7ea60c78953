"""Which continuations beam search's selection returns, and in which order, where totals tie or lie close: groups that the 64-bit totals
tell apart hold the same continuations, and inside a group those of one beam, and those of exactly equal totals, stand in order.

Totals are off by what a row's sum of exponentials in fp32 is: a few hundred terms after each other, (V / 4 / 512 + 40) 2^-24 of itself, so of its
logarithm; that is the same for every continuation of a beam.  The difference of a logit and its row's largest one, and its sum with the beam's
part, are in 64 bits: 2^-52 of the totals each."""
import math

import pytest
import torch

from seedplane_amd.beam import beam_select

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _totals(logits, scores):
    """Per beam the distance of each logit from its row's largest (exact in 64 bits for these types) and score - log sum exp."""
    x = logits.double().cpu()
    top = x.amax(-1, keepdim=True)
    below = x - top
    shift = scores.double().cpu().view(-1) - below.exp().sum(-1).log()
    return below, shift


def _check(logits, scores, n):
    B, K = scores.shape
    V = logits.shape[1]
    step = beam_select(logits, scores, n=n)
    below, shift = _totals(logits, scores)
    off = (V / 4 / 512 + 40) * 2.0 ** -24
    for b in range(B):
        rows = []
        for k in range(K):
            if not math.isfinite(float(scores[b, k])):
                continue
            d = below[b * K + k]
            order = torch.sort(d, descending=True, stable=True).indices[:n]
            rows += [(float(d[t] + shift[b * K + k]), k, int(t)) for t in order.tolist() if float(d[t]) > -math.inf]
        rows.sort(key=lambda r: (-r[0], r[1], r[2]))
        got = [(int(step.beams[b, i]), int(step.tokens[b, i])) for i in range(n)]
        m = min(n, len(rows))
        assert got[m:] == [(-1, -1)] * (n - m)
        got = got[:m]
        assert len(set(got)) == m
        # what must be among them, and what may: by totals at a distance from the n-th
        border = rows[m - 1][0]
        far = 2 * off + abs(border) * 2.0 ** -50
        must = {(k, t) for s, k, t in rows if s > border + far}
        may = {(k, t) for s, k, t in rows if s >= border - far}
        assert must <= set(got) <= may, b
        total = {(k, t): s for s, k, t in rows}
        for (k0, t0), (k1, t1) in zip(got, got[1:]):
            s0, s1 = total[k0, t0], total[k1, t1]
            assert s0 >= s1 - 2 * off - abs(s0) * 2.0 ** -50, (b, (k0, t0), (k1, t1))
        for k in range(K):                                   # one beam's stand by logit, then token, and are its best
            mine = [t for kk, t in got if kk == k]
            assert mine == [t for _, kk, t in rows if kk == k][:len(mine)], (b, k)
    return step


def _allowed(g, rows, V, count, dtype, fill):
    x = torch.full((rows, V), fill)
    at = torch.randperm(V, generator=g)[:count]
    x[:, at] = torch.randn((rows, count), generator=g) * 3
    return x.to(dtype)


@pytest.mark.parametrize('dtype', [F32, F16, BF16])
@pytest.mark.parametrize('V,n', [(300, 10), (20000, 20), (50257, 64)])
def test_grammars_by_the_lowest_value(gpu_device, dtype, V, n):
    """Three tokens allowed, the rest at the type's lowest value (fp32: totals at -3.4e38, whose differences only 64 bits hold apart)."""
    g = torch.Generator().manual_seed(V + n)
    x = _allowed(g, 3 * 5, V, 3, dtype, torch.finfo(dtype).min)
    step = _check(x.to(gpu_device), (-torch.rand((3, 5), generator=g) * 4).to(gpu_device), n)
    if dtype != F16:                                         # 2^128 holds no score beside it: all that are forbidden tie
        hidden = (x[0] == torch.finfo(dtype).min).nonzero()[:, 0].tolist()
        for b in range(3):
            assert step.beams[b, 15:].tolist() == [0] * max(0, n - 15) and step.tokens[b, 15:].tolist() == hidden[:max(0, n - 15)]


@pytest.mark.parametrize('dtype', [F32, F16, BF16])
@pytest.mark.parametrize('V,n', [(400, 6), (4096, 8), (30000, 40), (151936, 8)])
def test_ties_and_close_totals(gpu_device, dtype, V, n):
    """Few distinct logits, beams whose scores are equal, apart by a multiple of the logits' step, or by less than fp32 tells."""
    g = torch.Generator().manual_seed(V * 3 + n)
    x = torch.randint(-8, 9, (4 * 4, V), generator=g).float() / 4
    x[4:8] = x[4]                                            # a request whose beams have the same rows
    s = torch.tensor([[0.0, 0.0, -0.25, -0.5], [-1.0, -1.0, -1.25, -1.5], [-3.0, -3.0000002, -3.0000005, -7.0], [-0.1, -0.2, -0.3, -math.inf]])
    _check(x.to(dtype).to(gpu_device), s.to(gpu_device), n)


@pytest.mark.parametrize('V,n', [(257, 1), (300, 40), (511, 64), (512, 64), (2304, 33), (2500, 64)])
def test_parts_that_hold_more_than_the_buffer(gpu_device, V, n):
    """Rows, and last parts of rows, of 257 to 511 values, of which too few threads have one for a border: rising, falling, equal, random."""
    g = torch.Generator().manual_seed(V + n)
    line = torch.linspace(-3, 3, V)
    x = torch.stack([line, line.flip(0), torch.zeros(V), torch.randn(V, generator=g)])
    _check(x.to(gpu_device), torch.zeros((4, 1), device=gpu_device), n)
    _check(x.to(gpu_device), torch.tensor([[0.0, -0.3, -0.3, -2.0]], device=gpu_device), max(n, 4))


@pytest.mark.parametrize('where', [0, 3, 7])
def test_rows_whose_parts_are_mostly_masked(gpu_device, where):
    """One beam over 64 parts, of which a wave of the merge has only masked ones, or all others have: no border by first entries."""
    g = torch.Generator().manual_seed(where)
    V = 64 * 2048
    part = torch.arange(V) // 2048
    x = torch.randn((2, V), generator=g)
    x[0, part % 8 == where] = -math.inf
    x[1, part % 8 != where] = -math.inf
    for n in (1, 7, 16):
        _check(x.to(gpu_device), torch.zeros((2, 1), device=gpu_device), n)
