"""What an append without rotation writes into blocks is the definition's in every bit: scales are the fp32 quotient of the largest magnitude and
the largest code, codes the rounded fp32 quotient of value and scale, also where it lies next to a half."""
import pytest
import torch

from seedplane_amd.paged import PagedKV

pytestmark = pytest.mark.gpu

I8, E4M3 = torch.int8, torch.float8_e4m3fn
MOST = {I8: 127.0, E4M3: 448.0}


def _codes(q, cache):
    q = q.clamp(-MOST[cache], MOST[cache])
    return q.round().to(I8) if cache == I8 else q.to(E4M3)


def _halves(g, rows, heads, hd, cache, dtype):
    """Values near the middle of two codes of scales whose reciprocals are not exact: (c + 1/2) m / 127, the largest 127 m / 127."""
    most = torch.randint(1, 4000, (rows // 16, 1, heads, 1), generator=g).double() / 64
    c = torch.randint(-127, 127, (rows // 16, 16, heads, hd), generator=g).double() + 0.5
    x = c * most / 127 if cache == I8 else (torch.randint(-64, 64, c.shape, generator=g).double() + 0.5) * most / 64
    x[:, 0, :, 0] = most[:, 0, :, 0]
    return x.clamp(-most, most).view(rows, heads, hd).to(dtype)


@pytest.mark.parametrize('cache', [I8, E4M3])
@pytest.mark.parametrize('dtype', [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize('rows,heads,hd', [(16, 2, 64), (96, 4, 128), (48, 3, 24), (4160, 1, 64)])
def test_scales_and_codes(gpu_device, cache, dtype, rows, heads, hd):
    """Whole blocks of 16, then one position more of each with a larger value, by which the others are rounded once more."""
    g = torch.Generator().manual_seed(rows + hd)
    page = 32
    x, y = (_halves(g, rows, heads, hd, cache, dtype) for _ in range(2))
    kv = PagedKV.allocate(rows // 16, page, heads, hd, cache, scale_block=16)
    table = torch.arange(rows // 16, dtype=torch.int32, device=gpu_device).view(-1, 1)     # a sequence a block: the first half of its page
    seq = torch.arange(rows // 16, dtype=torch.int32, device=gpu_device).repeat_interleave(16)
    pos = torch.arange(16, dtype=torch.int32, device=gpu_device).repeat(rows // 16)
    order = torch.randperm(rows, generator=g)
    kv.append(x[order].to(gpu_device), y[order].to(gpu_device), seq[order.to(gpu_device)], pos[order.to(gpu_device)], table)

    def check(pool, scale, codes, want):
        assert torch.equal(scale[:, :, 0].cpu(), want)
        assert torch.equal(pool[:, :, :16].contiguous().view(torch.uint8).cpu(), codes.contiguous().view(torch.uint8))
    held = []
    for new, pool, scale in ((x, kv.k, kv.k_scale), (y, kv.v, kv.v_scale)):
        v = new.float().view(-1, 16, heads, hd).transpose(1, 2)            # [blocks, heads, 16, hd]
        s = v.abs().amax((-2, -1)) / torch.tensor(MOST[cache])
        codes = _codes(v / s[..., None, None], cache)
        check(pool, scale, codes, s)
        held.append((codes, s))
    more = torch.randint(0, 16, (rows // 16,), generator=g).clamp_min(1)
    z = [(2.7 * t.float().view(-1, 16, heads, hd).abs().amax(1) * torch.rand((rows // 16, heads, hd), generator=g)).to(dtype) for t in (x, y)]
    kv.append(z[0].to(gpu_device), z[1].to(gpu_device), torch.arange(rows // 16, dtype=torch.int32, device=gpu_device),
              more.int().to(gpu_device), table)
    for new, (codes, s), pool, scale in zip(z, held, (kv.k, kv.v), (kv.k_scale, kv.v_scale)):
        grown = torch.maximum(new.float().abs().amax(-1) / torch.tensor(MOST[cache]), s)
        kept = _codes(codes.float() * (s / grown)[..., None, None], cache)
        kept = kept.view(torch.uint8)
        kept[torch.arange(rows // 16), :, more] = _codes(new.float() / grown[..., None], cache).view(torch.uint8)
        check(pool, scale, kept.view(cache), grown)
