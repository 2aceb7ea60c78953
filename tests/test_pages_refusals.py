"""The page pool's and the beam selection's C entry points refuse bad arguments before any GPU call: the pointers here are never
dereferenced."""
import ctypes

import pytest

from pages_ref import Pages
from seedplane_amd import _lib

P = 1 << 20


def pool(**kw):
    d = _lib.PagePoolDesc(P, None, P, P, P, P, P, 4 * 16 * 64, 16 * 64, 64, 6, _lib.SP_DT_F16, 8, 16, 4, 64, 0, 5, 7, 1)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


BAD = [dict(pools=None), dict(table=None), dict(lengths=None), dict(holders=None), dict(missing=None), dict(workspace=None), dict(workspace=P + 8),
       dict(n_pools=0), dict(n_pools=65536), dict(dtype=_lib.SP_DT_F32), dict(dtype=7), dict(n_pages=0), dict(page_size=0), dict(n_kv_heads=0),
       dict(head_dim=0), dict(max_seqs=0), dict(max_seqs=65536), dict(max_pages=0), dict(max_seqs=60000, max_pages=60000), dict(page_stride=63),
       dict(head_stride=0), dict(row_stride=-64), dict(scale_block=16), dict(scales=P), dict(scales=P, scale_block=12), dict(scales=P, scale_block=-16),
       dict(page_size=1 << 20, n_kv_heads=1 << 10, head_stride=1 << 40), dict(max_pages=1 << 28, max_seqs=1)]


@pytest.mark.parametrize('kw', BAD)
def test_pools_are_refused(kw):
    lib, ref = _lib.load(), ctypes.byref(pool(**kw))
    for rc in (lib.sp_op_pages_fork(ref, P, None), lib.sp_op_pages_grow(ref, P, None), lib.sp_op_pages_free(ref, 2, P, None),
               lib.sp_op_pages_compact(ref, P, None), lib.sp_op_pages_copy(ref, 2, P, P, None)):
        assert rc == _lib.SP_EINVAL and lib.sp_last_error()


def test_arguments_are_refused():
    lib, ref = _lib.load(), ctypes.byref(pool())
    for rc in (lib.sp_op_pages_fork(None, P, None), lib.sp_op_pages_fork(ref, None, None), lib.sp_op_pages_grow(ref, None, None),
               lib.sp_op_pages_free(ref, -1, P, None), lib.sp_op_pages_free(ref, 1, None, None), lib.sp_op_pages_compact(None, None, None),
               lib.sp_op_pages_copy(ref, -1, P, P, None), lib.sp_op_pages_copy(ref, 1, None, P, None), lib.sp_op_pages_copy(ref, 1, P, None, None)):
        assert rc == _lib.SP_EINVAL
    assert lib.sp_op_pages_free(ref, 0, None, None) == _lib.SP_OK and lib.sp_op_pages_copy(ref, 0, None, None, None) == _lib.SP_OK
    assert lib.sp_pages_workspace(0, 1, 1) == 0 and lib.sp_pages_workspace(1, 1, 0) == 0
    for S, W, N in ((1, 1, 1), (128, 40, 5000), (65535, 16000, 1000000)):
        need = 64 + 4 * (S + S + 1 + S * W + 2 * N) + 12 * max(S, N)
        assert need <= lib.sp_pages_workspace(S, W, N) <= need + 6 * 16


def select(dtype=0, logits=P, ld=100, B=2, K=3, V=100, scores=P, n=6, n_eos=1, eos=True, ws=P, outs=(P,) * 6):
    ends = (ctypes.c_int32 * 8)() if eos else None
    return _lib.load().sp_op_beam_select(dtype, logits, ld, B, K, V, scores, n, n_eos, ends, *outs, ws, None)


@pytest.mark.parametrize('kw', [
    dict(dtype=3), dict(dtype=-1), dict(logits=None), dict(scores=None), dict(ws=None), dict(ws=P + 8), dict(ld=99), dict(B=-1), dict(K=0), dict(K=65, n=65),
    dict(V=0), dict(V=1 << 30, ld=1 << 30), dict(n=2), dict(n=65), dict(n_eos=-1), dict(n_eos=9), dict(eos=False), dict(B=30000),
    *(dict(outs=(P,) * i + (None,) + (P,) * (5 - i)) for i in range(6))])
def test_selections_are_refused(kw):
    assert select(**kw) == _lib.SP_EINVAL and _lib.load().sp_last_error()


def test_no_requests_is_no_call():
    assert select(B=0, logits=None, scores=None, ws=None, outs=(None,) * 6) == _lib.SP_OK
    lib = _lib.load()
    assert lib.sp_op_beam_select_workspace(0, 1, 1, 1) == 0 and lib.sp_op_beam_select_workspace(1, 4, 1000, 65) == 0
    for B, K, V, n in ((1, 1, 1, 1), (1, 4, 151936, 8), (32, 8, 151936, 16), (1, 64, 151936, 64), (1000, 64, 10, 64)):
        assert 0 < lib.sp_op_beam_select_workspace(B, K, V, n) <= B * K * 64 * (8 * n + 8)


def test_struct_layout_matches_c(tmp_path):
    import subprocess
    from pathlib import Path
    src = tmp_path / 'layout.c'
    names = [f for f, _ in _lib.PagePoolDesc._fields_]
    c = ['pools_dev', 'scales_dev', 'table_dev', 'lengths_dev', 'holders_dev', 'missing_dev', 'workspace_dev'] + names[7:]
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "seedplane_hip.h"\nint main(void) { printf("%zu", sizeof(sp_page_pool));'
                   + ''.join(f'printf(" %zu", offsetof(sp_page_pool, {f}));' for f in c) + ' return 0; }')
    exe = tmp_path / 'layout'
    subprocess.run(['gcc', '-std=c99', '-I', str(Path(__file__).resolve().parents[1] / 'include'), str(src), '-o', str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [ctypes.sizeof(_lib.PagePoolDesc)] + [getattr(_lib.PagePoolDesc, f).offset for f in names]


def test_rules_on_lists():
    """The lists that the GPU tests compare with, on a case worked by hand: pages of 4, sequences of 6, 4 and 1 positions."""
    p = Pages(6, 4, 3, 3)
    p.grow([6, 4, 1])
    assert p.table() == [[0, 1, -1], [2, -1, -1], [3, -1, -1]] and p.holders == [1, 1, 1, 1, 0, 0]
    p.fork([0, 0, 1])
    assert p.table() == [[0, 1, -1], [0, 3, -1], [2, -1, -1]] and p.copies == [(1, 3, 2)] and p.lengths == [6, 6, 4]
    assert p.holders == [2, 1, 1, 1, 0, 0]
    p.free([0])
    assert p.holders == [1, 0, 1, 1, 0, 0] and p.compact() == [0, 1, 2, 1, 4, 5] and p.table() == [[-1] * 3, [0, 1, -1], [2, -1, -1]]
    p.grow([9, 3, 20])
    assert p.missing == 4 and p.table() == [[3, 4, 5], [0, 1, -1], [2, -1, -1]] and p.lengths == [9, 9, 12]
