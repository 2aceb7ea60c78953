"""The plan of the paged attention (host code): its items read every position that a query sees exactly once for every K/V head,
nothing else, and every record has one writer."""
import ctypes

import numpy as np
import pytest

from seedplane_amd import _lib

ALL = 1 << 30


def plan(nh, nkv, q_lens, kv_lens, groups, hd=128):
    lib = _lib.load()
    q, kv = np.array(q_lens, np.int32), np.array(kv_lens, np.int32)
    g = np.array(groups if groups is not None else [], np.int32).reshape(-1, 2)
    size, shared = np.ascontiguousarray(g[:, 0]), np.ascontiguousarray(g[:, 1])
    toks = np.zeros((int(q.sum()), 8), np.int32)
    recs, n = ctypes.c_int64(), ctypes.c_int32()
    args = (nh, nkv, hd, len(q), q.ctypes.data, kv.ctypes.data, len(g), size.ctypes.data, shared.ctypes.data)
    _lib.check(lib.sp_attn_plan_items(*args, 0, None, ctypes.byref(n), None, ctypes.byref(recs)))
    items = np.zeros((n.value, 12), np.int32)
    _lib.check(lib.sp_attn_plan_items(*args, n.value, items.ctypes.data, ctypes.byref(n), toks.ctypes.data, None))
    return items, toks, recs.value


CASES = [
    (2, 1, [1], [1], None),
    (12, 2, [1] * 16, [2048 + 17 * i + 1 for i in range(16)], [(16, 2048)]),
    (28, 4, [1] * 5, [700, 1, 0, 64, 4097], [(1, 700), (1, 1), (1, 0), (2, 64)]),
    (28, 4, [9, 0, 3, 1], [300, 500, 203, 201], [(4, 200)]),
    (14, 2, [5, 5], [3, 9], [(2, 2)]),                       # queries in front of the first position; nothing can be shared
    (16, 16, [37, 100, 2], [137, 400, 102], [(2, 100), (1, 50)]),
    (32, 1, [3, 70], [1000, 1070], [(2, 999)]),
    (8, 8, [1, 1, 1], [0, 0, 0], None),
    (28, 4, [200, 300], [4296, 4396], [(2, 4096)]),
    (4, 4, [1] * 64, [33] * 64, [(64, 32)]),
    (12, 2, [1, 1], [100000, 100001], [(2, 99999)]),
    (12, 2, [0, 0], [5, 5], [(2, 3)]),
]


@pytest.mark.parametrize('hd', [64, 128])
@pytest.mark.parametrize('case', range(len(CASES)))
def test_every_seen_position_is_read_once_and_records_have_one_writer(case, hd):
    nh, nkv, q_lens, kv_lens, groups = CASES[case]
    G = nh // nkv
    items, toks, n_recs = plan(nh, nkv, q_lens, kv_lens, groups, hd)
    seqs = [s for s, n in enumerate(q_lens) for _ in range(n)]
    pos = [kv_lens[s] - q_lens[s] + i for s, n in enumerate(q_lens) for i in range(n)]
    group_of = []
    for g, (n, shared) in enumerate(groups or [(1, 0)] * len(q_lens)):
        group_of += [(g, shared)] * n
    read = {}
    writer = {}
    alone = set()
    for tok0, ntok, kvh, seq, k0, k1, pos0, rec, kind, *_ in items.tolist():
        assert 1 <= ntok * G <= 32 << kind and 0 <= kvh < nkv and 0 <= k0 < k1
        for i in range(ntok):
            t = tok0 + i
            end = min(k1, pos0 + i + 1)
            if pos0 == ALL:                             # shared positions, through another sequence's table
                g, shared = group_of[seqs[t]]
                assert group_of[seq] == (g, shared) and k1 <= shared and q_lens[seq] > 0 and k1 <= pos[t] + 1
                end = k1
            else:
                assert seq == seqs[t] and pos0 + i == pos[t] and k1 <= max(kv_lens[seq], 1)
            if end > k0:
                read.setdefault((t, kvh), []).append((k0, end))
            base, parts, tile, at = toks[t].reshape(4, 2)
            which = 0 if pos0 == ALL else 1
            if rec < 0:
                assert parts[which] == -1 and parts[1 - which] == 0 and (t, kvh) not in alone
                alone.add((t, kvh))
            else:
                assert parts[which] >= 1 and tile[which] == ntok and at[which] == i
                part = [j for j in range(parts[which])
                        if (base[which] + (kvh * parts[which] + j) * tile[which] + i) * G == rec + i * G]
                assert len(part) == 1
                key = rec + i * G
                assert key not in writer and key + G <= n_recs
                writer[key] = (t, kvh)
    for t, p in enumerate(pos):
        for kvh in range(nkv):
            at = 0
            for a, b in sorted(read.get((t, kvh), [])):
                assert a == at, (t, kvh, read[t, kvh])
                at = b
            assert at == max(0, p + 1)
            parts = toks[t][2:4]
            if parts[0] >= 0 and parts[1] >= 0:
                expect = {(int(toks[t][w]) + (kvh * int(parts[w]) + j) * int(toks[t][4 + w]) + int(toks[t][6 + w])) * G
                          for w in range(2) for j in range(parts[w])}
                assert all(writer[r] == (t, kvh) for r in expect)


def test_shared_positions_are_read_once_for_the_group():
    items, _, _ = plan(12, 2, [1] * 16, [2048 + 100] * 16, [(16, 2048)])
    shared = items[items[:, 6] == ALL]
    for h in range(2):
        assert (shared[shared[:, 2] == h][:, 5] - shared[shared[:, 2] == h][:, 4]).sum() == 2048
    own = items[items[:, 6] != ALL]
    assert (own[:, 4] >= 2048).all() and (own[:, 5] - own[:, 4]).sum() == 16 * 100 * 2


def test_records_stay_within_the_workspace():
    """The number of records never passes the bound that the workspace is made for."""
    rng = np.random.default_rng(0)
    for _ in range(200):
        nkv = int(rng.choice([1, 2, 4, 8]))
        G = int(rng.choice([1, 3, 6, 7, 8, 32]))
        n = int(rng.integers(1, 40))
        q = rng.integers(0, int(rng.choice([2, 10, 120])), n)
        kv = q + rng.integers(0, int(rng.choice([50, 3000, 60000])), n)
        shared = int(kv.min() * rng.choice([0, 0.5, 1]))
        items, toks, recs = plan(nkv * G, nkv, q.tolist(), kv.tolist(), [(n, shared)])
        rows = int(q.sum())
        assert recs <= 2 * rows * nkv * G + 2 * 512 * 128
        assert len(items) <= 2 * rows * nkv + 512


def test_bad_lengths_are_refused():
    def bad(q, kv, groups=None, nh=12, nkv=2):
        with pytest.raises(ValueError):
            plan(nh, nkv, q, kv, groups)
    bad([1], [-1])
    bad([1], [1 << 30])
    bad([1, 1], [10, 20], [(1, 5)])                          # the groups do not cover the sequences
    bad([1, 1], [10, 20], [(3, 5)])
    bad([1, 1], [10, 20], [(2, 11)])                         # a sequence shorter than the shared length
    bad([1, 1], [10, 20], [(2, -1)])
    bad([1, 1], [10, 20], [(0, 1), (2, 1)])
    bad([1], [1], nh=66, nkv=2)                              # 33 query heads per K/V head
    bad([1], [1], nh=5, nkv=2)
    lib = _lib.load()
    q = (ctypes.c_int32 * 1)(-1)
    n = ctypes.c_int32()
    one = (ctypes.c_int32 * 1)(1)
    items = (ctypes.c_int32 * 12)()
    call = lambda a, b, n_seq=1, cap=0, out=None, count=n: lib.sp_attn_plan_items(
        2, 1, 64, n_seq, a, b, 0, None, None, cap, out, None if count is None else ctypes.byref(count), None, None)
    assert call(one, one) == _lib.SP_OK and n.value == 1
    assert call(q, one) == _lib.SP_EINVAL and call(None, one) == _lib.SP_EINVAL and call(one, one, n_seq=0) == _lib.SP_EINVAL
    assert call(one, one, count=None) == _lib.SP_EINVAL
    assert call(one, one, out=items) == _lib.SP_ECAPACITY and call(one, one, cap=1, out=items) == _lib.SP_OK
