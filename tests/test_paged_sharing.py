"""What a group's plan reads of its shared positions: once per row tile for all sequences with queries, whichever others stand
between them."""
import numpy as np
import pytest

from test_paged_plan import ALL, plan


def positions_read(nh, nkv, q_lens, kv_lens, groups):
    """Positions that the items of K/V head 0 read, of all and of the shared items."""
    items, toks, _ = plan(nh, nkv, q_lens, kv_lens, groups)
    head = items[items[:, 2] == 0]
    length = head[:, 5] - head[:, 4]
    return int(length.sum()), int(length[head[:, 6] == ALL].sum())


@pytest.mark.parametrize('order', [[1, 0] * 16, [0, 1] * 16, [0] * 16 + [1] * 16, [1] * 16 + [0] * 16, [1] + [0] * 16 + [1] * 15])
@pytest.mark.parametrize('idle_kv', [8192 + 5, 0])
def test_idle_sequences_do_not_end_a_groups_sharing(order, idle_kv):
    """A sequence without queries, whatever its length, takes nothing from the group: the same reads as without it."""
    kv = [8192 + 7 if q else idle_kv for q in order]
    alone = positions_read(28, 4, [1] * 16, [8192 + 7] * 16, [(16, 8192)])
    assert alone == (8192 + 16 * 7, 8192)                    # 112 rows: one tile
    assert positions_read(28, 4, order, kv, [(32, 8192)]) == alone


def test_drafts_between_idle_sequences_share():
    q = [9, 0, 0, 3, 0, 1, 9]
    kv = [2000 + n for n in q]
    assert positions_read(12, 2, q, kv, [(7, 2000)]) == positions_read(12, 2, [9, 3, 1, 9], [2009, 2003, 2001, 2009], [(4, 2000)])
