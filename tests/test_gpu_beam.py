"""Beam search's selection on the GPU against the definition in 64 bits.

Scores: a row's sum of exponentials is taken in fp32, a few hundred terms after each other at most (here (V / 4 / 512 + 40) 2^-24 of
itself), its logarithm is off by as much, and a score is rounded once, 2^-24 of itself.  Order: exact within a beam; across beams where
totals differ by more than that."""
import math

import pytest
import torch

from seedplane_amd.beam import BeamStep, beam_select

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _reference(logits, scores, n, ends):
    """Per request: the list of (total, beam, token) of all its continuations that can be among the n best, in order."""
    B, K = scores.shape
    V = logits.shape[1]
    x = logits.double().cpu()
    dead = x.isnan().any(-1) | (x == math.inf).any(-1)
    # (x - log sum exp x, with the largest logit taken from x first: 64 bits lose it beside a type's lowest value)
    total = (torch.log_softmax(x, -1) + scores.double().cpu().view(-1, 1)).masked_fill((x == -math.inf) | dead[:, None], -math.inf).nan_to_num(nan=-math.inf, neginf=-math.inf)
    out = []
    for b in range(B):
        rows = []
        for k in range(K):
            t = total[b * K + k]
            order = torch.sort(t, descending=True, stable=True).indices[:n].tolist()
            rows += [(float(t[i]), k, i) for i in order if float(t[i]) > -math.inf]
        out.append(sorted(rows, key=lambda r: (-r[0], r[1], r[2]))[:n])
    return out


def _check(logits, scores, n=None, eos=None, out=None):
    ends = [] if eos is None else [eos] if isinstance(eos, int) else list(eos)
    B, K = scores.shape
    V = logits.shape[1]
    step = beam_select(logits, scores, n=n, eos=eos, out=out)
    n = step.scores.shape[1]
    off = (V / 4 / 512 + 40) * 2.0 ** -24
    want = _reference(logits, scores, n, ends)
    got = [x.cpu() for x in step]
    for b in range(B):
        w = want[b]
        mine = [(float(got[0][b, i]), int(got[1][b, i]), int(got[2][b, i])) for i in range(n)]
        assert mine[len(w):] == [(-math.inf, -1, -1)] * (n - len(w)), (b, mine, w)
        mine = mine[:len(w)]
        assert len(set((k, t) for _, k, t in mine)) == len(mine)
        gaps = [w[i][0] - w[i + 1][0] for i in range(len(w) - 1) if w[i][1] != w[i + 1][1]]
        if not gaps or min(gaps) > 2 * off or all(g == 0 or g > 2 * off for g in gaps) and len(set(s for s, _, _ in w)) == 1:
            assert [(k, t) for _, k, t in mine] == [(k, t) for _, k, t in w], b
        for (s, k, t), (total, _, _) in zip(mine, w):
            assert abs(s - total) <= off + abs(total) * 2.0 ** -24 + 1e-30, (b, s, total)
        going = [(s, b * K + k, t) for s, k, t in mine if t not in ends][:K]
        going += [(-math.inf, -1, -1)] * (K - len(going))
        assert [(float(got[3][b, i]), int(got[4][b, i]), int(got[5][b, i])) for i in range(K)] == going
    return step


def _inputs(g, B, K, V, dtype, dev, spread=2.5):
    x = torch.randn((B * K, V), generator=g) * spread
    x.scatter_add_(1, torch.randint(0, V, (B * K, min(V, 20)), generator=g), torch.rand((B * K, min(V, 20)), generator=g) * 10)
    return x.to(dtype).to(dev), (-torch.rand((B, K), generator=g) * 5).to(dev)


@pytest.mark.parametrize('dtype', [F32, F16, BF16])
@pytest.mark.parametrize('B,K,V,n,eos', [
    (1, 1, 1, None, None), (1, 1, 7, None, 3), (2, 3, 5, None, 0), (3, 4, 1000, None, 17), (1, 4, 151936, None, 5), (5, 8, 32001, 20, [1, 2]),
    (2, 32, 4097, None, 9), (1, 64, 2049, None, None), (1, 2, 50257, 64, [3, 4, 5]), (40, 8, 8191, None, 8), (7, 1, 4096, 1, None)])
def test_select(gpu_device, dtype, B, K, V, n, eos):
    print(f'beam {dtype} {B} {K} {V} {n} {eos}', flush=True)
    _check(*_inputs(torch.Generator().manual_seed(B * 31 + V), B, K, V, dtype, gpu_device), n=n, eos=eos)


@pytest.mark.parametrize('dtype', [F32, BF16])
def test_ends_first_steps_and_grammars(gpu_device, dtype):
    """The best tokens end; one beam lives; almost everything is forbidden, by -infinity or by the type's lowest value."""
    g = torch.Generator().manual_seed(2)
    x, s = _inputs(g, 4, 5, 20000, dtype, gpu_device)
    x[:, 77] = 30
    step = _check(x, s, eos=[77, 78])
    assert (step.tokens[:, 0] == 77).all() and not (step.next_tokens == 77).any()
    s[:, 1:] = -math.inf
    step = _check(x, s, eos=77)
    assert (step.beams == 0).all()
    s[1] = -math.inf
    s[2, 0] = math.nan
    step = _check(x, s, eos=77)
    assert (step.next_rows[1:3] == -1).all() and (step.scores[1:3] == -math.inf).all()
    x, s = _inputs(g, 4, 5, 20000, dtype, gpu_device)
    y = torch.full_like(x, -math.inf)
    keep = torch.randint(0, 20000, (3,), generator=g).to(gpu_device)
    y[:, keep] = x[:, keep]
    y[5:10] = -math.inf
    step = _check(y, s)
    assert (step.tokens[0] >= 0).all() and (step.tokens[1] == -1).all()
    y = torch.where(y == -math.inf, torch.finfo(dtype).min, y)
    _check(y, s, n=20)


@pytest.mark.parametrize('V', [9, 3000, 40000])
def test_ties_go_to_the_lowest(gpu_device, V):
    """Equal logits everywhere, few distinct values, equal beams, rising and falling rows (the buffer overflows)."""
    g = torch.Generator().manual_seed(V)
    s = torch.zeros((2, 4), device=gpu_device)
    flat = torch.zeros((8, V), device=gpu_device)
    step = _check(flat, s, n=min(8, V))
    assert step.tokens[0].tolist() == list(range(min(8, V))) and (step.beams == 0).all()
    few = torch.randint(0, 3, (8, V), generator=g).float().to(gpu_device)
    s2 = torch.tensor([[0.0, -0.5, -1.25, -7.0]], device=gpu_device).expand(2, 4).contiguous()
    _check(few, s2, n=min(8, V))
    _check(few.to(BF16), s2, n=min(8, V))
    rising = torch.linspace(-5, 5, V, device=gpu_device).expand(8, V)
    _check(rising.contiguous(), s2, n=min(40, 4 * V))
    _check(rising.flip(1).contiguous(), s2, n=min(40, 4 * V))


def test_bad_logits_and_extremes(gpu_device):
    g = torch.Generator().manual_seed(8)
    x, s = _inputs(g, 3, 4, 9000, F32, gpu_device)
    x[1, 8999], x[4, 0], x[6, 4500] = math.nan, math.inf, math.nan
    x[8:] *= 1000                                             # one token has all of the probability
    step = _check(x, s, n=16)
    assert not (step.beams[0] == 1).any() and not (step.beams[1] == 0).any() and not (step.beams[1] == 2).any()
    x[:] = math.nan
    assert (_check(x, s).next_rows == -1).all()


def test_rows_apart_unaligned_and_out(gpu_device):
    g = torch.Generator().manual_seed(9)
    x, s = _inputs(g, 2, 3, 5000, F16, gpu_device)
    want = _check(x, s, eos=1)
    wide = torch.full((6, 5003), 60.0, dtype=F16, device=gpu_device)
    wide[:, 1:5001] = x
    out = BeamStep.allocate(2, 3, 6, gpu_device)
    assert _check(wide[:, 1:5001], s, eos=1, out=out) is out
    assert all(torch.equal(a, b) for a, b in zip(out, want))
    none = beam_select(x[:0], s[:0], eos=1)
    assert none.scores.shape == (0, 6) and none.next_rows.shape == (0, 3)


def test_captured_and_on_another_stream(gpu_device):
    g = torch.Generator().manual_seed(10)
    x, s = _inputs(g, 3, 4, 30000, BF16, gpu_device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    tape = torch.cuda.CUDAGraph()
    with torch.cuda.graph(tape, stream=side):
        step = beam_select(x, s, eos=4)
    for _ in range(4):
        y, t = _inputs(g, 3, 4, 30000, BF16, gpu_device)
        x.copy_(y)
        s.copy_(t)
        tape.replay()
        want = beam_select(y, t, eos=4)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(step, want))
    with torch.cuda.stream(side):
        other = beam_select(x, s, eos=4)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(other, want))


def test_refusals(gpu_device):
    x, s = torch.zeros((6, 50), device=gpu_device), torch.zeros((2, 3), device=gpu_device)
    for bad in [dict(logits=x[0]), dict(logits=x.double()), dict(logits=x.T), dict(logits=x.cpu()), dict(scores=s.view(-1)), dict(scores=s.double()),
                dict(scores=s.cpu()), dict(scores=s[:1]), dict(scores=torch.zeros((3, 2), device=gpu_device).T), dict(n=2), dict(n=65),
                dict(eos=list(range(30))), dict(eos=[0] * 9, n=6), dict(out=BeamStep.allocate(2, 3, 4, gpu_device), n=5),
                dict(logits=x[:1].expand(6, 50))]:
        with pytest.raises(ValueError):
            beam_select(**{**dict(logits=x, scores=s), **bad})
