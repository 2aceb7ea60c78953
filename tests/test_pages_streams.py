"""What a page pool allocates for itself outlives its calls on other streams than the one it was made on."""
import pytest
import torch

from seedplane_amd import _lib, paged, pages


def test_memory_is_noted_for_the_stream_of_a_call(monkeypatch):
    """No GPU: the pool is host memory here, streams are numbers, the library's calls are left out."""
    kv = paged.PagedKV.__new__(paged.PagedKV)
    kv.k, kv.v = torch.zeros((6, 2, 32, 64), dtype=torch.int8), torch.zeros((6, 2, 32, 64), dtype=torch.int8)
    kv.k_scale, kv.v_scale, kv.scale_block = torch.zeros((6, 2, 2)), torch.zeros((6, 2, 2)), 16
    kv.device, kv.dtype, kv.lib = kv.k.device, kv.k.dtype, _lib.load()
    kv.n_pages, kv.n_kv_heads, kv.page_size, kv.head_dim = kv.k.shape
    now, noted = [7], []
    monkeypatch.setattr(pages, '_call', lambda *a: None)
    monkeypatch.setattr(paged, '_raw_stream', lambda i: now[0])
    monkeypatch.setattr(pages, '_raw_stream', lambda i: now[0], raising=False)
    monkeypatch.setattr(torch.cuda, 'current_stream', lambda device=None: f'stream {now[0]}')
    monkeypatch.setattr(torch.Tensor, 'record_stream', lambda self, stream: noted.append((self.data_ptr(), stream)))
    pool = pages.PagePool([kv], 3, 2)
    ints = lambda *x: torch.tensor(x, dtype=torch.int32)
    calls = [lambda: pool.fork(ints(0, 1, 2)), lambda: pool.grow(ints(1, 1, 1)), lambda: pool.free(ints(0)), lambda: pool.compact(),
             lambda: pool.copy(ints(0), ints(1))]
    own = {t.data_ptr() for t in (pool.table, pool.lengths, pool.holders, pool.missing, pool._workspace, pool._pools, pool._scales)}
    for i, call in enumerate(calls):
        now[0] = 7
        call()
        assert not noted
        now[0] = 8 + i
        call()
        assert own <= {p for p, s in noted if s == f'stream {8 + i}'}
        noted.clear()
        call()                                               # (once is enough)
        assert not noted


@pytest.mark.gpu
def test_memory_is_not_given_away_under_a_call(gpu_device):
    """A pool is dropped while its fork still waits on another stream: what is allocated meanwhile is other memory."""
    kv = paged.PagedKV.allocate(40, 16, 2, 64, torch.float16)
    pool = pages.PagePool([kv], 10, 6)
    counts, parents = (torch.tensor(x, dtype=torch.int32, device=gpu_device) for x in ([20] * 10, [0] * 10))
    pool.grow(counts)
    own = {t.data_ptr(): t.nbytes for t in (pool.table, pool.lengths, pool.holders, pool.missing, pool._workspace, pool._pools)}
    side, done = torch.cuda.Stream(), torch.cuda.Event()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(100_000_000)
        pool.fork(parents)
        done.record()
    del pool
    taken = [torch.empty(n, dtype=torch.uint8, device=gpu_device) for n in own.values() for _ in range(4)]
    assert not done.query()
    assert not own.keys() & {t.data_ptr() for t in taken}
    side.synchronize()
