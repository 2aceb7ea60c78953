"""Groups whose sequences with few queries stand between idle ones and long prompts: attention against 64-bit forms, and calls
captured with fewer rows than a later batch has."""
import pytest
import torch

from paged_ref import attend64, paged_batch
from seedplane_amd.paged import AttentionPlan, PagedKV
from test_gpu_paged import TYPES, _attend, _within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype,cache', TYPES)
@pytest.mark.parametrize('hd', [64, 128])
@pytest.mark.parametrize('q_lens,own,groups,nh,nkv,page', [
    ([1, 36, 1, 0, 18, 2], [3, 40, 70, 9, 18, 2], [(6, 96)], 28, 4, 16),
    ([0, 4, 1, 8, 0, 3, 1, 12], [0, 4, 300, 90, 5, 3, 33, 12], [(5, 700), (3, 64)], 32, 1, 4),
    ([1, 256, 70, 128, 1], [1, 300, 100, 128, 65], [(5, 320)], 4, 4, 32),
    ([1, 0] * 8, [9, 0] * 8, [(16, 1024)], 12, 2, 64),
])
def test_short_sequences_between_others(gpu_device, dtype, cache, hd, q_lens, own, groups, nh, nkv, page):
    print(f'groups {dtype} {cache} {hd} {q_lens} {own} {groups} {nh} {nkv}', flush=True)
    shared = [n for size, n in groups for _ in range(size)]
    _attend(gpu_device, q_lens, [a + b for a, b in zip(shared, own)], groups, nh, nkv, hd, page, dtype, cache, seed=hd)


@pytest.mark.parametrize('rows', [1, 37, 38, 56, 60])
def test_a_call_captured_with_fewer_rows(gpu_device, rows):
    """Rows within the captured call are the eager call's, the others are neither read nor written."""
    dtype = torch.bfloat16
    q_lens, kv_lens, groups = [1, 36, 1, 0, 18, 2], [1203, 1240, 1270, 1209, 1218, 1202], [(6, 1200)]
    g = torch.Generator().manual_seed(3)
    q, k, v, table, _ = paged_batch(g, q_lens, kv_lens, groups, 28, 4, 128, 16, dtype, dtype, gpu_device, rows_behind=4)
    kv, plan = PagedKV(k, v), AttentionPlan(28, 4, 128, 64, 6)
    plan.set(q_lens, kv_lens, groups)
    want = plan.run(q, kv, table)
    ref, _, bound = attend64(q[:58], k, v, table, q_lens, kv_lens, 128 ** -0.5)
    _within(want[:58], ref, bound)
    plan.set([1], [5])
    out = torch.full_like(q, 3.0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.run(q[:rows], kv, table, out=out[:rows])
    plan.set(q_lens, kv_lens, groups)
    for _ in range(3):
        out.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        n = min(rows, 58)
        _within(out[:n], ref[:n], bound[:n])
        assert (out[n:] == 3).all()


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
@pytest.mark.parametrize('hd', [64, 128])
@pytest.mark.parametrize('captured,later', [(0, 8000), (200, 8000), (8000, 1500), (8000, 300), (200, 700)])
def test_a_captured_call_has_the_eager_calls_bits(gpu_device, dtype, hd, captured, later):
    """Whatever lengths the plan held at the capture, empty ones too: few and many parts to join."""
    B, nh, nkv, page = 5, 14, 2, 16
    g = torch.Generator().manual_seed(later + hd)
    lens = [later + 3 * i for i in range(B)]
    q, k, v, table, _ = paged_batch(g, [1] * B, lens, None, nh, nkv, hd, page, dtype, dtype, gpu_device)
    wide = torch.full((B, 520), -1, dtype=torch.int32, device=gpu_device)
    wide[:, :table.shape[1]] = table
    kv, plan = PagedKV(k, v), AttentionPlan(nh, nkv, hd, B, B)
    plan.set([1 if captured else 0] * B, [captured] * B)
    out, lse = torch.zeros_like(q), torch.zeros(B, nh, device=gpu_device)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.run(q, kv, wide, out=out, lse=lse)
    plan.set([1] * B, lens)
    want_lse = torch.zeros_like(lse)
    want = plan.run(q, kv, wide, lse=want_lse)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(lse, want_lse)


def test_the_default_output_of_a_captured_call_has_zeros_behind_the_plans_rows(gpu_device):
    """Replays after the plan has got fewer rows than it had at the capture, and more again."""
    g = torch.Generator().manual_seed(8)
    q, k, v, table, _ = paged_batch(g, [1] * 6, [90, 700, 33, 64, 5, 210], None, 8, 2, 64, 16, torch.float16, torch.float16, gpu_device)
    kv, plan = PagedKV(k, v), AttentionPlan(8, 2, 64, 6, 6).set([1] * 6, [90, 700, 33, 64, 5, 210])
    want = plan.run(q, kv, table)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = plan.run(q, kv, table)
    for n in (6, 2, 5, 0, 6):
        plan.set([1] * n + [0] * (6 - n), [90, 700, 33, 64, 5, 210])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[:n], want[:n]) and (out[n:] == 0).all(), n


@pytest.mark.parametrize('page', [1, 3, 127, 4097, 65536, 70000])
def test_page_sizes_and_far_positions(gpu_device, page):
    """A position's page, for sizes below and above the positions read."""
    dtype, hd, n = torch.float16, 64, 66000
    g = torch.Generator().manual_seed(page)
    pages = -(-n // page)
    order = torch.randperm(pages, generator=g).int()
    pools = [torch.randn((pages, 1, page, hd), generator=g).to(dtype) for _ in range(2)]
    q = (torch.randn((3, 4, hd), generator=g) * 1.5).to(dtype)
    flat = [p[order.long()].reshape(1, 1, -1, hd) for p in pools]           # the positions in order: one page
    want, _, bound = attend64(q, *flat, torch.zeros((1, 1), dtype=torch.int32), [3], [n], hd ** -0.5)
    kv = PagedKV(*(p.to(gpu_device) for p in pools))
    got = AttentionPlan(4, 1, hd, 3, 1).set([3], [n]).run(q.to(gpu_device), kv, order.view(1, -1).to(gpu_device))
    _within(got, want, bound)
