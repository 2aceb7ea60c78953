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


def tokens_of(item, toks):
    """An item's tokens: a range, or from the first on those that have records of shared positions."""
    tok0, n = int(item[0]), int(item[1])
    if item[9] < 0:
        return list(range(tok0, tok0 + n))
    return [t for t in range(tok0, len(toks)) if toks[t][2] > 0][:n]


@pytest.mark.parametrize('nh,nkv,q_lens', [(28, 4, [1, 400] * 4), (28, 4, [400, 1, 0, 400, 1, 1]), (12, 2, [3, 128, 9, 0, 256, 1])])
def test_a_groups_order_does_not_matter(nh, nkv, q_lens):
    """Prompts that fill their own tiles stand between the short ones: the same reads as with the short ones first."""
    first = sorted(q_lens)
    kv = lambda lens: [8192 + n for n in lens]
    n = len(q_lens)
    want = positions_read(nh, nkv, first, kv(first), [(n, 8192)])
    per = 128 // (nh // nkv)                                 # tokens of a row tile; 128 tokens of 6 heads do not fill 7 of 21
    short = sum(q for q in q_lens if -(-q // per) * per * 8 > q * 9)
    assert want[1] == 8192 * -(-short // per)
    assert positions_read(nh, nkv, q_lens, kv(q_lens), [(n, 8192)]) == want


def test_random_groups_read_every_position_once():
    """Groups in any order of idle, short and filling sequences: each token reads its positions once, records have one writer."""
    rng = np.random.default_rng(5)
    for _ in range(60):
        nkv, G = int(rng.choice([1, 2])), int(rng.choice([1, 6, 7, 32]))
        q, kv, groups = [], [], []
        for _ in range(rng.integers(1, 4)):
            size, shared = int(rng.integers(1, 9)), int(rng.integers(0, 900))
            q += rng.choice([0, 1, 1, 2, 5, 18, 64, 126, 128, 200], size).tolist()
            kv += (shared + rng.integers(0, 300, size)).tolist()
            groups.append((size, shared))
        items, toks, recs = plan(nkv * G, nkv, q, kv, groups)
        seqs = np.repeat(np.arange(len(q)), q)
        pos = np.concatenate([np.arange(b - a, b) for a, b in zip(q, kv)]) if sum(q) else np.zeros(0, int)
        group = np.repeat(np.arange(len(groups)), [n for n, _ in groups])
        reads, writer = {}, {}
        for item in items:
            tok0, ntok, kvh, seq, k0, k1, pos0, rec = item[:8].tolist()
            tokens = tokens_of(item, toks)
            assert len(tokens) == ntok and tokens[0] == tok0
            which = 0 if pos0 == ALL else 1
            for i, t in enumerate(tokens):
                if which:
                    assert item[9] == -1 and seq == seqs[t] and pos0 + i == pos[t]
                else:
                    assert group[seq] == group[seqs[t]] and k1 <= groups[group[seq]][1] and k1 <= pos[t] + 1 and q[seq] > 0
                end = k1 if not which else min(k1, pos[t] + 1)
                if end > k0:
                    reads.setdefault((t, kvh), []).append((k0, end))
                base, parts, tile, at = toks[t].reshape(4, 2)[:, which]
                if rec < 0:
                    assert parts == -1 and which == 1
                    continue
                assert tile == ntok and at == i
                key = rec // G + i
                assert any(base + (kvh * parts + j) * tile + at == key for j in range(parts))
                assert (key not in writer) and (key + 1) * G <= recs
                writer[key] = t
        for t in range(len(pos)):
            for h in range(nkv):
                at = 0
                for a, b in sorted(reads.get((t, h), [])):
                    assert a == at
                    at = b
                assert at == max(0, pos[t] + 1)
