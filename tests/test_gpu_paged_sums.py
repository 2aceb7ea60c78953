"""Weighted sums are held in 32 bits from the products to the output, also where a row's keys are read in parts."""
import pytest
import torch

from paged_ref import attend64, paged_batch
from seedplane_amd.paged import AttentionPlan, PagedKV
from test_gpu_paged import TYPES, _within

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16

BATCHES = [                                                  # q_lens, kv_lens, groups
    ([1, 1, 1], [9000, 3000, 5000], None),
    ([1] * 12, [2048 + 9 * i + 1 for i in range(12)], [(12, 2048)]),
    ([9, 1, 20], [3009, 3001, 3020], [(3, 3000)]),
    ([70, 1], [1070, 300], None),
    ([1, 5], [300, 400], None),                              # not cut
]


@pytest.mark.parametrize('dtype,lowest', [(BF16, -60), (F16, -4)])
@pytest.mark.parametrize('hd', [64, 128])
@pytest.mark.parametrize('batch', range(len(BATCHES)))
def test_columns_keep_their_bits_beside_larger_ones(gpu_device, dtype, lowest, hd, batch):
    """Values of a column times a power of two give outputs times that power, in every bit: a product by 2^n commutes with every
    rounding short of the types' least values, whatever the other columns hold."""
    q_lens, kv_lens, groups = BATCHES[batch]
    g = torch.Generator().manual_seed(hd + batch)
    q, k, v, table, _ = paged_batch(g, q_lens, kv_lens, groups, 12, 2, hd, 8, dtype, dtype, gpu_device)
    v *= 64
    plan = AttentionPlan(12, 2, hd, sum(q_lens), len(q_lens)).set(q_lens, kv_lens, groups)
    size = torch.exp2(torch.linspace(0, lowest, hd, device=gpu_device).round()).to(dtype)
    want = plan.run(q, PagedKV(k, v), table) * size
    got = plan.run(q, PagedKV(k, v * size), table)
    # (outputs below fp16's normal range round to its least step instead)
    normal = want.abs() >= torch.finfo(dtype).tiny
    assert torch.equal(got[normal], want[normal]) and normal.float().mean() > 0.99


@pytest.mark.parametrize('dtype,cache', TYPES)
@pytest.mark.parametrize('hd', [64, 128])
@pytest.mark.parametrize('batch', range(len(BATCHES)))
def test_parts_round_no_more_than_whole_ranges(gpu_device, dtype, cache, hd, batch):
    """The 64-bit form's bound without its term for parts kept in fewer bits: that term is 2^-12 + 2^-20 of the row's largest sum of
    weighted magnitudes, which is the same form over the values' magnitudes."""
    q_lens, kv_lens, groups = BATCHES[batch]
    g = torch.Generator().manual_seed(7 * hd + batch)
    q, k, v, table, scales = paged_batch(g, q_lens, kv_lens, groups, 12, 2, hd, 8, dtype, cache, gpu_device)
    plan = AttentionPlan(12, 2, hd, sum(q_lens), len(q_lens)).set(q_lens, kv_lens, groups)
    got = plan.run(q, PagedKV(k, v, *scales), table)
    args = (table, q_lens, kv_lens, hd ** -0.5, *scales)
    want, _, bound = attend64(q, k, v, *args)
    if dtype == BF16:
        bound = bound - attend64(q, k, v.float().abs(), *args)[0].amax(-1, keepdim=True) * (2.0 ** -12 + 2.0 ** -20)
    _within(got, want, bound)
