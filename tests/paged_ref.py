"""Plain 64-bit forms of the paged operators, and inputs for their tests."""
import math

import numpy as np
import torch

HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float8_e4m3fn: 2.0 ** -4}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -133, torch.float8_e4m3fn: 2.0 ** -10}


def rotate64(x, pos, inv, factor, rot, layout):
    """x [rows, heads, hd] (any type) rotated in 64 bits on the CPU."""
    y = x.detach().double().cpu().clone()
    a = pos.cpu().double()[:, None] * inv
    c, s = (a.cos() * factor)[:, None], (a.sin() * factor)[:, None]
    one, two = (slice(0, rot // 2), slice(rot // 2, rot)) if layout == 'half' else (slice(0, rot, 2), slice(1, rot, 2))
    p, q = y[..., one].clone(), y[..., two].clone()
    y[..., one], y[..., two] = p * c - q * s, q * c + p * s
    return y


def rotate_bound(x, rot, layout, factor, out_dtype, want):
    """Most that a rotated value may be off: the reduced turn t in [-1, 1] is rounded to 32 bits (2^-25, times pi), sincospif is
    good to 2 steps of a value up to 1 (2^-23), the factor, the two products and their sum round once each (4 x 2^-24): below
    2^-21 of (|x1| + |x2|) factor; then half a step of the output type."""
    y = x.detach().double().cpu().abs()
    size = torch.zeros_like(y)
    one, two = (slice(0, rot // 2), slice(rot // 2, rot)) if layout == 'half' else (slice(0, rot, 2), slice(1, rot, 2))
    size[..., one] = size[..., two] = (y[..., one] + y[..., two]) * factor
    return size * 2.0 ** -21 + (want.abs() + size * 2.0 ** -21) * HALF[out_dtype] + TINY[out_dtype]


def attend64(q, k, v, table, q_lens, kv_lens, scale, k_scale=None, v_scale=None):
    """(out, lse, bound) in 64 bits on the CPU for a paged batch.  Entries outside the pool hide their positions.

    bound, per output value, of a kernel with 32-bit sums whose weights are rounded to q's type before their product with
    V: scores carry (hd + 4) roundings of their absolute sum and the exponent's argument and exp2 a few of their own, so a
    weight is off by e^d - 1 <= 2 d of itself (the weights' sum likewise); rounding a weight costs half a step, or the
    type's smallest half step where it is subnormal; the sum over n keys n 2^-24; the output half a step.  Where a bf16 row's
    keys are read in parts, a part's outputs are kept as fp16 shares of its largest: a share of at most 1 is off by 2^-12, its
    scaling there and back by a few 2^-24, and the parts' largest, joined by their weights, are at most the row's largest sum of
    weighted magnitudes."""
    n_pages, nkv, page, hd = k.shape
    nh, half = q.shape[1], HALF[q.dtype]
    out = torch.zeros(q.shape, dtype=torch.float64)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64)
    bound = torch.zeros(q.shape, dtype=torch.float64)
    kd, vd, qd = k.float().cpu().double(), v.float().cpu().double(), q.double().cpu()
    if k_scale is not None:
        kd = kd * k_scale.cpu().double()[:, None, None]
        vd = vd * v_scale.cpu().double()[:, None, None]
    tab = table.cpu().numpy()
    r0 = 0
    for s, (nq, n) in enumerate(zip(q_lens, kv_lens)):
        at = np.arange(n)
        pages = tab[s][at // page] if n else np.zeros(0, int)
        ok = (pages >= 0) & (pages < n_pages)
        at, pages = at[ok], pages[ok]
        keys, vals = kd[pages, :, at % page], vd[pages, :, at % page]          # [n, nkv, hd]
        for i in range(nq):
            see = int((at <= n - nq + i).sum())
            if see:
                kk, vv = keys[:see].repeat_interleave(nh // nkv, 1), vals[:see].repeat_interleave(nh // nkv, 1)
                qr = qd[r0 + i]
                sc = (qr[None] * kk).sum(-1) * scale                            # [see, nh]
                size = (qr.abs()[None] * kk.abs()).sum(-1) * scale
                w = torch.softmax(sc, 0)
                out[r0 + i] = (w[..., None] * vv).sum(0)
                lse[r0 + i] = torch.logsumexp(sc, 0)
                d = size.amax(0) * (hd + 4) * 2.0 ** -24 + (sc.abs().amax(0) + 4) * 2.0 ** -22
                A = (w[..., None] * vv.abs()).sum(0)
                # a weight relative to the largest of its part (1); the sum of a part's weights is at least 1
                small = see * TINY[q.dtype] * vv.abs().amax(0)
                bound[r0 + i] = A * (4 * d[:, None] + half + see * 2.0 ** -24 + 2.0 ** -22) + small + \
                    (out[r0 + i].abs() + A * half) * half + TINY[q.dtype] + \
                    (A.amax(-1, keepdim=True) * (2.0 ** -12 + 2.0 ** -20) if q.dtype == torch.bfloat16 else 0)
        r0 += nq
    return out, lse, bound


def paged_batch(g, q_lens, kv_lens, groups, nh, nkv, hd, page, dtype, cache, device, spare=5, rows_behind=0, stride=None, fill='nan'):
    """q, k, v (pools), table, scales for a batch; every pool row that no sequence holds is NaN (or `fill`), entries past a
    sequence's last page lie outside the pool."""
    rng = np.random.default_rng(int(torch.randint(0, 1 << 30, (1,), generator=g)))
    B = len(q_lens)
    need = [-(-n // page) for n in kv_lens]
    width = max(1, max(need)) + 1
    table = np.full((B, width), 1 << 30, np.int32)
    common, s = [], 0
    total = 0
    plan = []
    for size, shared in (groups or [(1, 0)] * B):
        whole = shared // page
        assert shared % page == 0                            # sequences have whole pages in common
        plan.append((s, size, whole, total))
        total += whole
        s += size
    firsts = []
    for s0, size, whole, at in plan:
        for s in range(s0, s0 + size):
            firsts.append((s, whole, at, total))
            total += max(0, need[s] - whole)
    order = rng.permutation(total + spare).astype(np.int32)
    n_pages = max(1, total + spare)
    if total + spare == 0:
        order = np.zeros(1, np.int32)
    for s, whole, at, mine in firsts:
        w = min(whole, need[s])
        table[s, :w] = order[at:at + w]
        table[s, w:need[s]] = order[mine:mine + need[s] - w]
    e4m3 = cache == torch.float8_e4m3fn
    scales = (None, None)
    if e4m3:
        scales = tuple(((torch.rand(nkv, generator=g) + 0.5) * 0.01).to(device) for _ in range(2))
    pools = []
    held = np.zeros((n_pages, page), bool)
    for s, n in enumerate(kv_lens):
        p = np.arange(n)
        held[table[s][p // page], p % page] = True
    held = torch.from_numpy(held)
    for i in range(2):
        x = torch.randn((n_pages, nkv, page, hd), generator=g)
        if i == 0:
            x = x + 0.5 * torch.randn((1, nkv, 1, hd), generator=g)
        x = x / scales[i].cpu()[:, None, None] if e4m3 else x
        x = x.clamp(-448, 448) if e4m3 else x
        x[~held.unsqueeze(1).expand(-1, nkv, -1)] = math.nan if fill == 'nan' else fill
        if stride:
            wide = torch.zeros((n_pages, stride), dtype=cache, device=device)
            wide[:, :nkv * page * hd] = x.reshape(n_pages, -1).to(cache).to(device)
            pools.append(wide[:, :nkv * page * hd].view(n_pages, nkv, page, hd) if n_pages > 1 else x.to(cache).to(device))
        else:
            pools.append(x.to(cache).to(device))
    q = (torch.randn((sum(q_lens) + rows_behind, nh, hd), generator=g) * 1.5).to(dtype).to(device)
    return q, pools[0], pools[1], torch.from_numpy(table).to(device), scales
