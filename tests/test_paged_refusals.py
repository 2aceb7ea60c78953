"""The paged operators' C entry points refuse bad arguments before any GPU call: the pointers here are never dereferenced."""
import ctypes

import pytest

from seedplane_amd import _lib

P = 1 << 20                                                    # an aligned address that is no memory


def rotary(inv=P, rot=64, layout=0):
    return _lib.RotaryDesc(inv, rot, layout, 1.0, 0)


def cache(dtype=_lib.SP_DT_F16, k=P, v=2 * P, ks=None, vs=None, stride=4 * 16 * 64, head=16 * 64, row=64, n=8, page=16, nkv=4, hd=64):
    return _lib.PagedKVDesc(k, v, ks, vs, stride, head, row, dtype, n, page, nkv, hd, 0)


def rotate(r=None, dtype=_lib.SP_DT_F16, rows=4, heads=8, hd=64, x=P, x_row=512, x_head=64, out=4 * P, out_row=512, out_head=64, pos=P):
    r = rotary() if r is None else r
    return _lib.load().sp_op_rotate(ctypes.byref(r) if r else None, dtype, rows, heads, hd, x, x_row, x_head, out, out_row, out_head,
                                    pos, None)


@pytest.mark.parametrize('kw', [
    dict(r=False), dict(dtype=3), dict(dtype=-1), dict(rows=-1), dict(heads=0), dict(hd=1), dict(hd=2048), dict(heads=1024),
    dict(r=rotary(inv=None)), dict(r=rotary(rot=63)), dict(r=rotary(rot=0)), dict(r=rotary(rot=66)), dict(r=rotary(layout=2)),
    dict(x=None), dict(out=None), dict(pos=None),
    dict(out=P + 128),                                          # overlaps, not in place
    dict(out=P, out_row=1024),                                  # the same memory with other strides
    dict(out_row=0), dict(out_head=0), dict(out_row=511), dict(out_row=-512), dict(out_head=32),
])
def test_rotate_refusals(kw):
    assert rotate(**kw) == _lib.SP_EINVAL
    assert _lib.load().sp_last_error()


def test_no_rows_is_no_call():
    assert rotate(rows=0, x=None, out=None, pos=None) == _lib.SP_OK
    assert append(rows=0, k=None, v=None, seq=None) == _lib.SP_OK


def append(kv=None, r=None, dtype=_lib.SP_DT_F16, rows=4, heads=8, q=8 * P, q_row=1024, k=9 * P, k_row=256, v=10 * P, pos=P, seq=P,
           at=P, table=P, n_seq=2, width=4, q_out=12 * P, q_dt=_lib.SP_DT_F16, qo_row=512, qo_head=64):
    kv = cache() if kv is None else kv
    r = rotary() if r is None else r
    return _lib.load().sp_op_paged_append(ctypes.byref(kv) if kv else None, ctypes.byref(r) if r else None, dtype, rows, heads, q, q_row, 64,
                                          k, k_row, 64, v, 256, 64, pos, seq, at, table, n_seq, width, q_out, q_dt, qo_row, qo_head, None)


@pytest.mark.parametrize('kw', [
    dict(kv=False), dict(kv=cache(k=None)), dict(kv=cache(v=None)), dict(kv=cache(dtype=_lib.SP_DT_F32)), dict(kv=cache(dtype=9)),
    dict(kv=cache(n=0)), dict(kv=cache(page=0)), dict(kv=cache(nkv=0)), dict(kv=cache(hd=0)), dict(kv=cache(stride=63)), dict(kv=cache(head=0)),
    dict(kv=cache(row=-64)), dict(kv=cache(row=32)),
    dict(kv=cache(ks=P, vs=P)), dict(kv=cache(dtype=_lib.SP_DT_E4M3)), dict(kv=cache(dtype=_lib.SP_DT_E4M3, ks=P)),
    dict(dtype=_lib.SP_DT_E4M3), dict(rows=-1), dict(heads=0), dict(heads=2000), dict(q_out=None), dict(q=None),
    dict(q_dt=_lib.SP_DT_E4M3), dict(n_seq=0), dict(width=0), dict(r=rotary(rot=128)),
    dict(k=None), dict(v=None), dict(seq=None), dict(at=None), dict(table=None), dict(pos=None),
    dict(q_out=8 * P, qo_row=1024, q_dt=_lib.SP_DT_F32),        # in place with another type
    dict(kv=cache(k=P, v=P)), dict(kv=cache(stride=1 << 62)), dict(kv=cache(row=1 << 57)),
    dict(k=P + 1024), dict(v=2 * P), dict(q=P), dict(q_out=2 * P + 4096), dict(k=P - 128),
    dict(q_out=9 * P), dict(q_out=10 * P + 64), dict(q_out=8 * P + 64), dict(qo_row=0), dict(qo_head=0),
])
def test_append_refusals(kw):
    assert append(**kw) == _lib.SP_EINVAL
    assert _lib.load().sp_last_error()


def test_plan_refusals():
    lib = _lib.load()
    h = ctypes.c_void_p()
    ok = (12, 2, 128, 16, 16)
    for i, bad in [(0, 0), (0, 13), (1, 0), (2, 96), (2, 0), (3, 0), (4, 0), (4, 65536), (3, 1 << 24), (0, 66), (0, 131072)]:
        a = list(ok)
        a[i] = bad
        assert lib.sp_attn_plan_create(*a, ctypes.byref(h)) == _lib.SP_EINVAL and not h.value, (i, bad)
    assert lib.sp_attn_plan_create(*ok, None) == _lib.SP_EINVAL
    one = (ctypes.c_int32 * 1)(1)
    assert lib.sp_attn_plan_set(None, 1, one, one, 0, None, None, None) == _lib.SP_EINVAL
    assert lib.sp_attn_plan_workspace(None) == 0
    lib.sp_attn_plan_destroy(None)
    kv = cache()
    assert lib.sp_op_paged_attention(None, ctypes.byref(kv), 1, 1, P, 512, 64, P, 1, 1, 1.0, P, 512, 64, None, P, None) == _lib.SP_EINVAL


def test_struct_layouts_match_c(tmp_path):
    import subprocess
    from pathlib import Path
    src = tmp_path / 'layout.c'
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "seedplane_hip.h"\nint main(void) {'
                   'printf("%zu %zu %zu %zu %zu %zu\\n", sizeof(sp_rotary), offsetof(sp_rotary, factor), sizeof(sp_paged_kv),'
                   'offsetof(sp_paged_kv, page_stride), offsetof(sp_paged_kv, dtype), offsetof(sp_paged_kv, head_dim)); return 0; }')
    exe = tmp_path / 'layout'
    include = Path(__file__).resolve().parents[1] / 'include'
    subprocess.run(['gcc', '-std=c99', '-I', str(include), str(src), '-o', str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    R, K = _lib.RotaryDesc, _lib.PagedKVDesc
    assert got == [ctypes.sizeof(R), R.factor.offset, ctypes.sizeof(K), K.page_stride.offset, K.dtype.offset, K.head_dim.offset]


def test_lengths_are_integers_in_range():
    import numpy as np
    from seedplane_amd.paged import _lengths
    assert _lengths([], 'x').tolist() == [] and _lengths([3, 0], 'x').dtype == np.int32
    assert _lengths(np.array([1 << 20], np.int64), 'x').tolist() == [1 << 20]
    for bad in ([1.5], [-1], [1 << 30], np.array([(1 << 32) + 5]), ['1'], [True]):
        with pytest.raises(ValueError):
            _lengths(bad, 'x')
