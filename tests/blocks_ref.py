"""Plain 64-bit forms of the operators over caches whose codes have a scale per block of positions and head."""
import math

import numpy as np
import torch

from paged_ref import HALF, TINY

MOST = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def dense64(codes, scale):
    """Codes [pages, heads, page, hd] and scales [pages, heads, blocks] as 64-bit values on the CPU."""
    c = codes.cpu()
    c = c.float().double()
    per = scale.shape[2]
    return (c.unflatten(2, (per, -1)) * scale.cpu().double()[..., None, None]).flatten(2, 3)


def append64(codes, scale, new, seq, at, table, page):
    """What an append of new [rows, heads, hd] (64-bit values, NaN-free) leaves: (values, scales, bound on the values), values and
    bounds NaN where a begun block's other positions are undefined.

    A new value is off by half a step of its code: half a scale (int8), 2^-4 of itself or 2^-10 of the scale (e4m3), and so is
    what a grown scale rounds once more; the scale and its reciprocal, and their products, are rounded 4 times (2^-22 of a value)."""
    cache, block = codes.dtype, codes.shape[2] // scale.shape[2]
    n_pages, n_seq, width = codes.shape[0], *table.shape
    val, sc = dense64(codes, scale), scale.cpu().double().clone()
    bound = torch.zeros_like(val)
    groups = {}
    for r, (s, p) in enumerate(zip(seq.tolist(), at.tolist())):
        if 0 <= s < n_seq and p >= 0 and p // page < width and 0 <= int(table[s, p // page]) < n_pages:
            groups.setdefault((int(table[s, p // page]), p % page // block), []).append((p % page, r))

    def step(x, s):
        if cache == torch.int8:
            return s * 0.5 + x.abs() * 2.0 ** -22
        return x.abs() * (2.0 ** -4 + 2.0 ** -22) + s * 2.0 ** -10
    for (e, b), rows in groups.items():
        part = slice(b * block, (b + 1) * block)
        begun = any(p % block == 0 for p, _ in rows)
        old = torch.zeros_like(sc[e, :, b]) if begun else sc[e, :, b]
        x = torch.stack([new[r] for _, r in rows])
        grown = torch.maximum((x.abs().amax((0, 2)) / MOST[cache]).clamp(2.0 ** -60, 2.0 ** 60), old)
        if begun:
            val[e, :, part], bound[e, :, part] = math.nan, math.nan
        else:
            for h in range(len(grown)):
                if grown[h] > old[h]:
                    bound[e, h, part] = step(val[e, h, part], grown[h])
        for p, r in sorted(rows, key=lambda t: t[1]):
            top = grown * MOST[cache]
            v = torch.minimum(torch.maximum(new[r], -top[:, None]), top[:, None])
            val[e, :, p] = v
            bound[e, :, p] = step(v, grown[:, None])
        sc[e, :, b] = grown
    return val, sc, bound


def attend_blocks64(q, k, ks, v, vs, table, q_lens, kv_lens, scale):
    """(out, lse, bound) in 64 bits for a paged batch over block scales.

    bound: as for other caches (paged_ref.attend64), with these differences.  A score's exponent carries the logarithm of its values'
    scale: the logarithm, its sum with the score and the scale's reciprocal in the weights' sum are off by a few 2^-24 of (|score| +
    |log2 scale| + 1), in a weight.  The product of weight and scale over the row's largest one is rounded to q's type: half a step of
    itself, or the type's smallest half step of that largest product, for each key, times the largest code."""
    n_pages, nkv, page, hd = k.shape
    nh, half = q.shape[1], HALF[q.dtype]
    out = torch.zeros(q.shape, dtype=torch.float64)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64)
    bound = torch.zeros(q.shape, dtype=torch.float64)
    kd, vd, qd = dense64(k, ks), dense64(v, vs), q.double().cpu()
    block = page // vs.shape[2]
    vsd = vs.cpu().double().repeat_interleave(block, 2)                          # [pages, nkv, page]
    tab = table.cpu().numpy()
    r0 = 0
    for s, (nq, n) in enumerate(zip(q_lens, kv_lens)):
        at = np.arange(n)
        pages = tab[s][at // page] if n else np.zeros(0, int)
        ok = (pages >= 0) & (pages < n_pages)
        at, pages = at[ok], pages[ok]
        keys, vals, vsc = kd[pages, :, at % page], vd[pages, :, at % page], vsd[pages, :, at % page]
        g = nh // nkv
        keys, vals, vsc = (x.repeat_interleave(g, 1) for x in (keys, vals, vsc))
        for i in range(nq):
            see = int((at <= n - nq + i).sum())
            if not see:
                continue
            kk, vv, vc, qr = keys[:see], vals[:see], vsc[:see], qd[r0 + i]
            sc = (qr[None] * kk).sum(-1) * scale
            size = (qr.abs()[None] * kk.abs()).sum(-1) * scale
            w = torch.softmax(sc, 0)
            out[r0 + i] = (w[..., None] * vv).sum(0)
            lse[r0 + i] = torch.logsumexp(sc, 0)
            d = size.amax(0) * (hd + 4) * 2.0 ** -24 + (sc.abs().amax(0) + vc.log2().abs().amax(0) + 4) * 2.0 ** -21
            A = (w[..., None] * vv.abs()).sum(0)
            most = 127.0 if k.dtype == torch.int8 else 448.0
            small = see * TINY[q.dtype] * (w * vc).amax(0)[:, None] * most
            bound[r0 + i] = A * (4 * d[:, None] + half + see * 2.0 ** -24 + 2.0 ** -22) + small + (out[r0 + i].abs() + A * half) * half + TINY[q.dtype]
        r0 += nq
    return out, lse, bound


def coded(x, cache, block):
    """Values [pages, heads, page, hd] as codes and scales, each block at its full range."""
    b = x.unflatten(2, (-1, block))
    scale = (b.abs().amax((-2, -1)) / MOST[cache]).float().clamp_min(1e-9)
    b = b / scale[..., None, None]
    return (b.round().to(torch.int8) if cache == torch.int8 else b.to(torch.float8_e4m3fn)).flatten(2, 3), scale.contiguous()
