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
