"""Paged K/V cache operators on MI355X: rotary embedding, append, and attention over pages with shared prefixes.

For servers that hold their K/V in pages rather than in `Qwen2Engine`'s rings, and for other models than Qwen2: rotary layouts
and scaled position tables, fp16 / bf16 / e4m3 / int8 caches, head ratios up to 32.  A page holds `page_size` positions of one
sequence for every K/V head; a table (int32 [sequences, most pages]) names each sequence's pages in order.  Sequences that
start with the same tokens may name the same pages, and `AttentionPlan` then reads those once for all of them:

    rotary = Rotary.from_config(config)                     # 'rope_scaling' honoured
    kv = PagedKV.allocate(n_pages, 64, kv_heads, head_dim)  # one layer's pages
    plan = AttentionPlan(heads, kv_heads, head_dim, max_rows=256, max_seqs=256)
    # one step: the plan once, then for every layer
    plan.set(q_lens, kv_lens, groups=[(sequences, shared_positions), ...])
    q = kv.append(k, v, seq, pos, table, rotary=rotary, q=q)
    out = plan.run(q, kv, table)

Every call runs on torch's current stream of its tensors' device, allocates nothing on the device except outputs that are not
given, and may be captured into a graph (`AttentionPlan.set` may not; a captured `run` follows later `set` calls).  The
reference has none of this (its cache is one tensor per sequence, seedplane/qwen_engine.py:18-29); the operators generalise
its _rope, cache copy and attention (qwen_engine.py:94-103, 121-135).
"""
import ctypes
import math
import weakref

import numpy as np
import torch

from . import _lib

_DTYPES = {torch.float32: _lib.SP_DT_F32, torch.float16: _lib.SP_DT_F16, torch.bfloat16: _lib.SP_DT_BF16,
           torch.float8_e4m3fn: _lib.SP_DT_E4M3, torch.int8: _lib.SP_DT_I8}
_INT32 = torch.int32
_CODES = (torch.float8_e4m3fn, torch.int8)
_FLOATS = {t: code for t, code in _DTYPES.items() if t not in _CODES}


def rotary_frequencies(rot_dim, theta=10000.0, scaling=None, length=None):
    """Angle per position of the rot_dim / 2 pairs (float64 tensor) and the factor on cosines and sines, for a
    `rope_scaling` entry of a Hugging Face config.json: rope_type (or type) 'default', 'linear', 'dynamic' (NTK: for `length`
    positions), 'yarn' or 'llama3' with their usual keys."""
    if rot_dim < 2 or rot_dim % 2:
        raise ValueError('rot_dim must be even and positive')
    j = torch.arange(0, rot_dim, 2, dtype=torch.float64)
    inv = 1.0 / theta ** (j / rot_dim)
    s = scaling or {}
    kind = s.get('rope_type') or s.get('type') or 'default'
    if kind == 'default':
        return inv, 1.0
    if kind not in ('linear', 'dynamic', 'yarn', 'llama3'):
        raise ValueError(f'unknown rope scaling {kind!r}')

    def value(key):
        if s.get(key) is None:
            raise ValueError(f'{kind} scaling needs {key}')
        return float(s[key])
    factor = value('factor')
    if not 1 <= factor < math.inf:
        raise ValueError('the scaling factor must be at least 1')
    if kind == 'linear':
        return inv / factor, 1.0
    original = s.get('original_max_position_embeddings')
    if not original:
        raise ValueError(f'{kind} scaling needs original_max_position_embeddings')
    if kind == 'dynamic':
        if rot_dim < 4:
            raise ValueError('dynamic scaling needs rot_dim of at least 4')
        grown = max(length or original, original)
        base = theta * (factor * grown / original - (factor - 1)) ** (rot_dim / (rot_dim - 2))
        return 1.0 / base ** (j / rot_dim), 1.0
    turns = original * inv / (2 * math.pi)                  # turns of each pair over the original length
    if kind == 'llama3':
        low, high = value('low_freq_factor'), value('high_freq_factor')
        if not low < high:
            raise ValueError('low_freq_factor must be less than high_freq_factor')
        keep = ((turns - low) / (high - low)).clamp(0, 1)   # 1: short waves, kept; 0: long ones, slowed by the factor
        return inv * (keep + (1 - keep) / factor), 1.0
    # YaRN: kept above beta_fast turns, slowed below beta_slow, a ramp over the pair's index between
    def index_at(n):
        return rot_dim * math.log(original / (n * 2 * math.pi)) / (2 * math.log(theta))
    lo, hi = index_at(s.get('beta_fast') or 32), index_at(s.get('beta_slow') or 1)
    if s.get('truncate', True):
        lo, hi = math.floor(lo), math.ceil(hi)
    lo, hi = max(lo, 0), min(hi, rot_dim - 1)
    slowed = ((torch.arange(rot_dim // 2, dtype=torch.float64) - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
    def grade(m):
        return 1.0 if factor <= 1 else 0.1 * m * math.log(factor) + 1.0
    attention = s.get('attention_factor')
    if attention is None:
        m, m_all = s.get('mscale'), s.get('mscale_all_dim')
        attention = grade(m) / grade(m_all) if m and m_all else grade(1)
    return inv * (1 - slowed) + inv / factor * slowed, float(attention)


_raw_stream, _current = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice
_is_capturing = torch._C._cuda_isCurrentStreamCapturing


def _device(device):
    d = torch.device('cuda' if device in ('hip', None) else device)
    if d.type != 'cuda':
        raise ValueError('seedplane_amd runs on a ROCm GPU device ("cuda"/"hip")')
    return torch.device('cuda', torch.cuda.current_device() if d.index is None else d.index)


def _call(fn, device, *args):
    """One library call on the current stream of `device`, with that device current."""
    i = device.index
    if _current() == i:
        rc = fn(*args, _raw_stream(i))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, _raw_stream(i))
    if rc:
        _lib.check(rc)


def _capturing(device):
    """Whether the current stream of `device` is being captured."""
    if _current() == device.index:
        return _is_capturing()
    with torch.cuda.device(device):
        return _is_capturing()


def _heads(x, name, device, heads, hd):
    """(dtype code, rows, row stride, head stride, address) of a [rows, heads, hd] tensor; heads None: any number."""
    dt, s, n = _FLOATS.get(x.dtype), x.stride(), x.shape
    if dt is None or x.device != device or len(n) != 3 or n[2] != hd or s[2] != 1 or (heads is not None and n[1] != heads):
        raise ValueError(f'{name} must be an fp32, fp16 or bf16 tensor [rows, {"heads" if heads is None else heads}, {hd}] on '
                         f'{device}, the values of a head side by side; got {x.dtype} {tuple(n)} with strides {s} on {x.device}')
    return dt, n[0], s[0], s[1], x.data_ptr()


def _ints(x, name, device, n):
    """The address of a contiguous int32 GPU tensor of n entries."""
    if x.dtype is not _INT32 or x.device != device or x.dim() != 1 or x.numel() != n or not x.is_contiguous():
        raise ValueError(f'{name} must be a contiguous int32 tensor on {device} with one entry per row')
    return x.data_ptr()


def _table(x, device):
    if x.dtype != torch.int32 or x.device != device or x.dim() != 2 or not x.is_contiguous() or not x.numel():
        raise ValueError(f'table must be a contiguous int32 tensor [sequences, most pages] on {device}')
    return x.data_ptr()


def _lengths(x, name):
    """Host integers as int32."""
    a = np.asarray(x)
    if a.size == 0:
        a = a.astype(np.int32)
    if a.dtype.kind not in 'iu' or (a.size and (a.min() < 0 or a.max() >= 1 << 30)):
        raise ValueError(f'{name} must be integers in [0, 2^30)')
    return np.ascontiguousarray(a, dtype=np.int32)


class Rotary:
    """A rotary position table on a device: `layout` 'half' (pairs j, j + rot_dim/2) or 'interleaved' (2j, 2j + 1), over the
    first `rot_dim` values of a head (default: all)."""

    def __init__(self, head_dim, theta=10000.0, rot_dim=None, layout='half', scaling=None, length=None, device='cuda'):
        if layout not in ('half', 'interleaved'):
            raise ValueError("layout must be 'half' or 'interleaved'")
        self.head_dim, self.rot_dim, self.layout = int(head_dim), int(head_dim if rot_dim is None else rot_dim), layout
        if self.rot_dim > self.head_dim:
            raise ValueError('rot_dim exceeds head_dim')
        self.inv_freq, self.factor = rotary_frequencies(self.rot_dim, theta, scaling, length)
        _lib.require_gpu()
        self.lib = _lib.load()
        self.device = _device(device)
        self._inv = self.inv_freq.to(self.device)
        self._stream = _raw_stream(self.device.index)
        self.desc = _lib.RotaryDesc(self._inv.data_ptr(), self.rot_dim,
                                    _lib.SP_ROPE_HALF if layout == 'half' else _lib.SP_ROPE_INTERLEAVED, self.factor, 0)
        self._ref = ctypes.addressof(self.desc)

    def _used(self):
        """The table's memory is given back only after the calls on this stream."""
        if _raw_stream(self.device.index) != self._stream:
            self._inv.record_stream(torch.cuda.current_stream(self.device))

    @classmethod
    def from_config(cls, config, layout='half', length=None, device='cuda'):
        """From a Hugging Face config.json dictionary (rope_theta, rope_scaling or rope_parameters, partial_rotary_factor)."""
        hd = config.get('head_dim') or config['hidden_size'] // config['num_attention_heads']
        p = config.get('rope_parameters') or {}
        scaling = config.get('rope_scaling') or (p if p.get('rope_type', 'default') != 'default' else None)
        if scaling and not scaling.get('original_max_position_embeddings'):
            scaling = dict(scaling, original_max_position_embeddings=config.get('max_position_embeddings'))
        parts = [x for x in (config.get('partial_rotary_factor'), p.get('partial_rotary_factor'), 1.0) if x is not None]
        rot = int(hd * parts[0])
        return cls(hd, config.get('rope_theta', p.get('rope_theta', 10000.0)), rot, layout, scaling, length, device)

    def apply(self, x, positions, out=None):
        """x [rows, heads, head_dim] rotated at int32 `positions` [rows] (any sign; with factor 1, negated positions undo the
        rotation and give its gradient).  `out` may be x."""
        dt, rows, row, head, addr = _heads(x, 'x', self.device, None, self.head_dim)
        pos = _ints(positions, 'positions', self.device, rows)
        if out is None:
            out = torch.empty_like(x)
            o_row, o_head, _ = out.stride()
            o_addr = out.data_ptr()
        elif out.shape != x.shape or out.dtype != x.dtype:
            raise ValueError('out must have the shape and type of x')
        else:
            _, _, o_row, o_head, o_addr = _heads(out, 'out', self.device, None, self.head_dim)
        _call(self.lib.sp_op_rotate, self.device, self._ref, dt, rows, x.shape[1], self.head_dim, addr, row, head, o_addr, o_row,
              o_head, pos)
        self._used()
        return out


class PagedKV:
    """One layer's pages: `k` and `v` [n_pages, kv_heads, page_size, head_dim], fp16, bf16, float8_e4m3fn or int8, or views of that
    shape (`pool.transpose(1, 2)` of a [n_pages, page_size, kv_heads, head_dim] pool, halves of one allocation, ...) with the
    same strides for both and the values of a row side by side.  A cache of 8 bits holds value / scale, with fp32 scales: [kv_heads]
    (e4m3), or for each block of positions [n_pages, kv_heads, page_size / block] (int8 or e4m3; blocks of 16 to 128 positions, whole
    16s), which `append` writes from the values themselves."""

    _lease = None                 # of an engine's pool (Qwen2Engine.paged_kv): what holds and dates its memory

    def __init__(self, k, v, k_scale=None, v_scale=None):
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or k.device != v.device or k.stride() != v.stride():
            raise ValueError('k and v must be [n_pages, kv_heads, page_size, head_dim] of one shape, type, device and layout')
        if k.dtype not in _DTYPES or k.dtype == torch.float32:
            raise ValueError('the cache must be fp16, bf16, float8_e4m3fn or int8')
        n, nkv, page, hd = k.shape
        if 0 in k.shape or k.stride(3) != 1 or any(m > 1 and s < hd for m, s in zip(k.shape[:3], k.stride())):
            raise ValueError('the values of a row must lie side by side and rows must not overlap')
        codes, self.scale_block = k.dtype in _CODES, 0
        for s in (k_scale, v_scale):
            if (s is not None) != codes:
                raise ValueError('a cache of 8 bits has k_scale and v_scale, others have none')
            if s is None:
                continue
            if s.dtype != torch.float32 or s.device != k.device or not s.is_contiguous() or s.shape != k_scale.shape:
                raise ValueError('scales must be contiguous fp32 tensors of one shape on the device of the cache')
            if s.dim() == 3 and s.shape[:2] == (n, nkv) and s.shape[2] and page % s.shape[2] == 0:
                self.scale_block = page // s.shape[2]
                if self.scale_block % 16 or self.scale_block > 128:
                    raise ValueError('blocks of a scale must be of 16, 32, .. 128 positions')
            elif s.shape != (nkv,) or k.dtype == torch.int8:
                raise ValueError('scales must be [kv_heads] (e4m3) or [n_pages, kv_heads, page_size / block]')
        _lib.require_gpu()
        self.lib = _lib.load()
        self.device = k.device
        if self.device.type != 'cuda':
            raise ValueError('seedplane_amd runs on a ROCm GPU device ("cuda"/"hip")')
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.n_pages, self.n_kv_heads, self.page_size, self.head_dim = n, nkv, page, hd
        self.dtype = k.dtype
        self.desc = _lib.PagedKVDesc(k.data_ptr(), v.data_ptr(), k_scale.data_ptr() if codes else None,
                                     v_scale.data_ptr() if codes else None, *self._strides(), _DTYPES[k.dtype], n, page, nkv, hd,
                                     self.scale_block)
        self._ref = ctypes.addressof(self.desc)

    def _strides(self):
        """Strides of pages, heads and rows; of a dimension of one entry: any that suits the kernels."""
        return [s if n > 1 else self.head_dim for n, s in zip(self.k.shape[:3], self.k.stride())]

    def _check_lease(self, table):
        """An engine's pool is where it was when this cache was made, and a table that Qwen2Engine.page_table gave is of it."""
        self._lease.check()
        made_for = getattr(table, '_lease', None)
        if made_for is not None and made_for != self._lease.key:
            raise ValueError('the page table is of an older pool, another engine or other pages: call page_table() again')

    @classmethod
    def allocate(cls, n_pages, page_size, n_kv_heads, head_dim, dtype=torch.float16, k_scale=None, v_scale=None, device='cuda',
                 scale_block=None):
        """Cleared pages; scale_block: positions of a block, whose scales are allocated too."""
        shape, device = (n_pages, n_kv_heads, page_size, head_dim), _device(device)
        if scale_block is not None:
            if scale_block < 1 or page_size % scale_block:
                raise ValueError('scale_block must divide page_size')
            if k_scale is not None or v_scale is not None:
                raise ValueError('scales of blocks are allocated here')
            k_scale, v_scale = (torch.zeros((n_pages, n_kv_heads, page_size // scale_block), device=device) for _ in range(2))
        return cls(torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device), k_scale, v_scale)

    def append(self, k, v, seq, pos, table, rotary=None, q=None, q_out=None, rotary_pos=None):
        """New tokens into the pages: row r's keys and values k[r], v[r] [kv_heads, head_dim] at position pos[r] of sequence
        seq[r] (int32 [rows]; a row with seq -1, or whose position has no page, writes nothing).  With `rotary` the keys turn by
        rotary_pos (default: pos) on the way, and the queries q [rows, heads, head_dim] into q_out (default: a new tensor of q's
        type; may be q itself), which is returned."""
        if self._lease is not None:
            self._check_lease(table)
        dev, nkv, hd = self.device, self.n_kv_heads, self.head_dim
        dt, rows, k_row, k_head, k_addr = _heads(k, 'k', dev, nkv, hd)
        v_dt, v_rows, v_row, v_head, v_addr = _heads(v, 'v', dev, nkv, hd)
        if v_dt != dt or v_rows != rows:
            raise ValueError('k and v must have the same rows and type')
        s, p, t = _ints(seq, 'seq', dev, rows), _ints(pos, 'pos', dev, rows), _table(table, dev)
        turn = p if rotary_pos is None else _ints(rotary_pos, 'rotary_pos', dev, rows)
        if rotary is not None and (rotary.head_dim != hd or rotary.device != dev):
            raise ValueError('the rotary table is of another head_dim or device')
        if q is not None:
            q_dt, q_rows, q_row, q_head, q_addr = _heads(q, 'q', dev, None, hd)
            if q_dt != dt or q_rows != rows:
                raise ValueError('q must have the rows and the type of k')
            if q_out is None:
                q_out = torch.zeros_like(q)                    # rows that write nothing
            elif q_out.shape != q.shape:
                raise ValueError('q_out must have the shape of q')
            o_dt, _, o_row, o_head, o_addr = _heads(q_out, 'q_out', dev, None, hd)
            queries, turned, nh = (q_addr, q_row, q_head), (o_addr, o_dt, o_row, o_head), q.shape[1]
        elif q_out is not None:
            raise ValueError('q_out without q')
        else:
            queries, turned, nh = (None, 0, 0), (None, 0, 0, 0), 0
        if rows:
            _call(self.lib.sp_op_paged_append, dev, self._ref, None if rotary is None else rotary._ref, dt, rows, nh, *queries,
                  k_addr, k_row, k_head, v_addr, v_row, v_head, turn, s, p, t, table.shape[0], table.shape[1], *turned)
            if rotary is not None:
                rotary._used()
        return q_out


    def read(self, seq, pos, table, dtype=torch.float16, out=None):
        """Keys and values at positions pos[r] of sequences seq[r] (int32 [rows]) as dense tensors [rows, kv_heads, head_dim] of
        `dtype` (fp32, fp16 or bf16), or into out, a pair of such; zeros where a row has no place."""
        if self._lease is not None:
            self._check_lease(table)
        dev, nkv, hd = self.device, self.n_kv_heads, self.head_dim
        if seq.dim() != 1:
            raise ValueError('seq must be [rows]')
        rows = seq.shape[0]
        s, p, t = _ints(seq, 'seq', dev, rows), _ints(pos, 'pos', dev, rows), _table(table, dev)
        if out is None:
            dt = _FLOATS.get(dtype)
            if dt is None:
                raise ValueError('dtype must be fp32, fp16 or bf16')
            k, v = torch.empty((2, rows, nkv, hd), dtype=dtype, device=dev).unbind(0)
            k_row, k_head, k_addr = nkv * hd, hd, k.data_ptr()
            v_row, v_head, v_addr = k_row, k_head, v.data_ptr()
        else:
            k, v = out
            dt, k_rows, k_row, k_head, k_addr = _heads(k, 'k', dev, nkv, hd)
            v_dt, v_rows, v_row, v_head, v_addr = _heads(v, 'v', dev, nkv, hd)
            if v_dt != dt or k_rows != rows or v_rows != rows:
                raise ValueError('out must be two tensors of one type, a row for each of seq')
        if rows:
            _call(self.lib.sp_op_paged_read, dev, self._ref, dt, rows, s, p, t, table.shape[0], table.shape[1], k_addr, k_row, k_head,
                  v_addr, v_row, v_head)
        return k, v


class AttentionPlan:
    """Attention over pages for batches of up to `max_rows` query tokens of up to `max_seqs` sequences; head_dim 64 or 128."""

    def __init__(self, n_heads, n_kv_heads, head_dim, max_rows, max_seqs, device='cuda'):
        _lib.require_gpu()
        self.lib = _lib.load()
        self.device = _device(device)
        self.n_heads, self.n_kv_heads, self.head_dim = int(n_heads), int(n_kv_heads), int(head_dim)
        self.max_rows, self.max_seqs = int(max_rows), int(max_seqs)
        h = ctypes.c_void_p()
        with torch.cuda.device(self.device):
            _lib.check(self.lib.sp_attn_plan_create(self.n_heads, self.n_kv_heads, self.head_dim, self.max_rows, self.max_seqs,
                                                    ctypes.byref(h)))
        self.h = h
        self._finalizer = weakref.finalize(self, self.lib.sp_attn_plan_destroy, h)
        self._ws = torch.empty(self.workspace_bytes, dtype=torch.uint8, device=self.device)
        self._ws_addr = self._ws.data_ptr()
        self._scale = 1.0 / math.sqrt(self.head_dim)
        self.rows = 0

    @property
    def workspace_bytes(self):
        """Bytes of a workspace for run(): calls that overlap each other need one each."""
        return int(self.lib.sp_attn_plan_workspace(self.h))

    def set(self, q_lens, kv_lens, groups=None):
        """The next batch (host integers): sequence s has q_lens[s] query tokens, the last of its kv_lens[s] cached positions.
        The tables replace those of the set before: runs on other streams that read them must have ended (or be waited for).
        groups: (sequences, shared positions) of each run of sequences whose tables name the same pages for their first positions,
        in any order and with idle ones (q_lens 0) among them; None: nothing is shared."""
        q, kv = _lengths(q_lens, 'q_lens'), _lengths(kv_lens, 'kv_lens')
        if q.ndim != 1 or q.shape != kv.shape:
            raise ValueError('q_lens and kv_lens must have one entry per sequence')
        size = shared = None
        n = 0
        if groups is not None:
            g = _lengths(groups, 'groups').reshape(-1, 2)
            size, shared, n = np.ascontiguousarray(g[:, 0]), np.ascontiguousarray(g[:, 1]), len(g)
            if n == 0 and len(q):
                raise ValueError('the groups do not cover the sequences')
        _call(self.lib.sp_attn_plan_set, self.device, self.h, len(q), q.ctypes.data, kv.ctypes.data, n,
              None if size is None else size.ctypes.data, None if shared is None else shared.ctypes.data)
        self.rows = int(q.sum())
        return self

    def run(self, q, kv, table, out=None, lse=None, scale=None, workspace=None):
        """Attention of q [rows, heads, head_dim] (fp16 or bf16) over the pages of `kv`; returns `out` (default: a new tensor,
        zeros behind the plan's rows; in a capture behind those of each replay).  lse: fp32 [rows, heads], filled with the
        logarithm of each row's sum of exponentials."""
        if kv._lease is not None:
            kv._check_lease(table)
        dev = self.device
        dt, rows, q_row, q_head, q_addr = _heads(q, 'q', dev, self.n_heads, self.head_dim)
        if kv.device != dev:
            raise ValueError('the cache is on another device')
        t = _table(table, dev)
        if out is None:
            # (a graph's replays may have fewer rows than the capture: they fill the rest anew)
            out = torch.empty_like(q) if rows == self.rows and not _capturing(dev) else torch.zeros_like(q)
            o_row, o_head, _ = out.stride()
            o_addr = out.data_ptr()
        elif out.shape != q.shape or out.dtype != q.dtype:
            raise ValueError('out must have the shape and type of q')
        else:
            _, _, o_row, o_head, o_addr = _heads(out, 'out', dev, self.n_heads, self.head_dim)
        if lse is not None and (lse.shape != q.shape[:2] or lse.dtype != torch.float32 or lse.device != dev
                                or not lse.is_contiguous()):
            raise ValueError('lse must be a contiguous fp32 [rows, heads] tensor')
        if workspace is None:
            ws = self._ws_addr
        else:
            if workspace.device != dev or not workspace.is_contiguous() or workspace.nbytes < self._ws.nbytes:
                raise ValueError('the workspace is too small or on another device')
            ws = workspace.data_ptr()
        _call(self.lib.sp_op_paged_attention, dev, self.h, kv._ref, dt, rows, q_addr, q_row, q_head, t, table.shape[0],
              table.shape[1], self._scale if scale is None else float(scale), o_addr, o_row, o_head,
              None if lse is None else lse.data_ptr(), ws)
        return out
