"""Pages of sequences on MI355X: which sequence holds which page of a model's paged caches, kept and changed on the device.

    caches = [PagedKV.allocate(n_pages, 64, kv_heads, head_dim, torch.int8, scale_block=16) for _ in range(layers)]
    pool = PagePool(caches, max_seqs=128, max_pages=64)
    pool.grow(counts)                                       # pages for new positions (int32 [max_seqs])
    caches[0].append(k, v, seq, pos, pool.table, ...)       # its table is the operators' page table
    pool.fork(parents)                                      # sequences continue others: beams, samples of one prompt
    pool.free(seqs)                                         # sequences end
    pool.compact()                                          # held pages move to the front

A fork shares full pages and copies the rows of a last page that is not full, in every layer, so no sequence ever writes what another
reads.  Every call runs on torch's current stream of the caches' device without waiting for it, allocates nothing and may be captured
into a graph; calls on one pool follow each other (a stream other than the one it was made on waits for that first).  The reference has
one tensor per sequence (seedplane/qwen_engine.py:18-29).
"""
import ctypes

import torch

from . import _lib
from .paged import _DTYPES, _call, _ints, _raw_stream


class PagePool:
    """The pages of `caches` (a PagedKV, or a list of them: the layers, alike in all but their memory) and `max_seqs` sequences of up to
    `max_pages` pages.  Where pages lie on each other, and over an engine's rings (Qwen2Engine.paged_kv), whose pages belong to its own
    caches, there are none to give: such a pool only copies, other calls raise ValueError.

    Tensors, which a program may read between calls: table int32 [max_seqs, max_pages] (-1 behind a sequence's pages), lengths int32
    [max_seqs], holders int32 [n_pages] (how many table entries name a page; add 1 to keep one that no sequence holds), missing int32
    [1] (pages that were wanted and not found, whose positions are hidden, and sequences cut at the table's width)."""

    def __init__(self, caches, max_seqs, max_pages):
        caches = list(caches) if isinstance(caches, (list, tuple)) else [caches]
        if not caches:
            raise ValueError('a pool needs a cache')
        kv = caches[0]
        alike = lambda c: (c.k.shape, c.dtype, c.device, tuple(c._strides()), c.scale_block)
        if any(alike(c) != alike(kv) for c in caches):
            raise ValueError('the caches must have one shape, type, device, layout and scale block')
        self.lib, self.device = kv.lib, kv.device
        self.caches, self.max_seqs, self.max_pages = caches, int(max_seqs), int(max_pages)
        self._leases = [c._lease for c in caches if c._lease is not None]      # of an engine's pool, which may move
        if not 1 <= self.max_seqs <= 65535 or self.max_pages < 1 or self.max_seqs * self.max_pages >= 1 << 30:
            raise ValueError('max_seqs must be in [1, 65535], max_pages positive and their product below 2^30')
        ints = lambda *shape: torch.zeros(shape, dtype=torch.int32, device=self.device)
        self.table = ints(self.max_seqs, self.max_pages).fill_(-1)
        self.lengths, self.holders, self.missing = ints(self.max_seqs), ints(kv.n_pages), ints(1)
        self._workspace = torch.zeros(self.lib.sp_pages_workspace(self.max_seqs, self.max_pages, kv.n_pages), dtype=torch.uint8,
                                      device=self.device)
        pools = [p.data_ptr() for c in caches for p in (c.k, c.v)]
        self._pools = torch.tensor(pools, dtype=torch.int64, device=self.device)
        self._scales = None
        if kv.scale_block:
            self._scales = torch.tensor([s.data_ptr() for c in caches for s in (c.k_scale, c.v_scale)], dtype=torch.int64, device=self.device)
        self.desc = _lib.PagePoolDesc(self._pools.data_ptr(), None if self._scales is None else self._scales.data_ptr(), self.table.data_ptr(),
                                      self.lengths.data_ptr(), self.holders.data_ptr(), self.missing.data_ptr(), self._workspace.data_ptr(),
                                      *kv._strides(), len(pools), _DTYPES[kv.dtype], kv.n_pages, kv.page_size, kv.n_kv_heads, kv.head_dim,
                                      kv.scale_block, self.max_seqs, self.max_pages, all(p % 16 == 0 for p in pools))
        self._ref = ctypes.addressof(self.desc)
        self._streams = {_raw_stream(self.device.index)}       # that the pool's memory is noted for
        self._memory = [t for t in (self.table, self.lengths, self.holders, self.missing, self._workspace, self._pools, self._scales)
                        if t is not None]

    def _run(self, fn, *args):
        for lease in self._leases:
            lease.check()
        raw = _raw_stream(self.device.index)
        if raw not in self._streams:
            # (given back only after the calls on this stream; a tensor keeps its streams for good)
            stream = torch.cuda.current_stream(self.device)
            for t in self._memory:
                t.record_stream(stream)
            self._streams.add(raw)
        _call(fn, self.device, self._ref, *args)
        return self

    def _give(self, fn, *args):
        if self._leases:
            raise ValueError("the pages are of an engine's rings: a pool over them can only copy")
        return self._run(fn, *args)

    def fork(self, parents):
        """Sequence s continues parents[s] (int32 [max_seqs]: any sequence, itself included; -1: s ends)."""
        return self._give(self.lib.sp_op_pages_fork, _ints(parents, 'parents', self.device, self.max_seqs))

    def grow(self, counts):
        """counts[s] more positions for each sequence (int32 [max_seqs]), with pages for them; they are the caller's to write.  To take
        positions back (rejected drafts) lower `lengths`, not into pages that other sequences hold too; the pages behind go with the next
        growth over them, fork or end."""
        return self._give(self.lib.sp_op_pages_grow, _ints(counts, 'counts', self.device, self.max_seqs))

    def free(self, seqs):
        """Sequences seqs (int32 [n]) end; their pages are free unless others hold them."""
        n = seqs.numel()
        return self._give(self.lib.sp_op_pages_free, n, _ints(seqs, 'seqs', self.device, n))

    def compact(self, places=None):
        """Held pages move to the lowest places.  places: int32 [n_pages], filled with each page's place afterwards."""
        return self._give(self.lib.sp_op_pages_compact, None if places is None else _ints(places, 'places', self.device, self.holders.numel()))

    def copy(self, src, dst):
        """Pages src[i] to dst[i] (int32 [n]) in every cache, with their scales; pairs outside the pool are left out.  A page is not a
        destination twice, nor both a source and a destination."""
        n = src.numel()
        return self._run(self.lib.sp_op_pages_copy, n, _ints(src, 'src', self.device, n), _ints(dst, 'dst', self.device, n))
