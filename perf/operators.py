"""Serving operators around a paged K/V cache, as cases that can be timed and checked one by one: the rotary embedding
(`rotate`), appending keys and values to the pages with the rotation on the way (`append`), and attention over the pages for a
batch whose sequences share a prefix (`attend`).

Head shapes are those of the Qwen2-0.5B / 1.5B / 7B presets (14/2 heads of 64, 12/2 of 128, 28/4 of 128) except where a case
says otherwise.  A page holds the rows of one sequence for all K/V heads: pools are [pages, kv_heads, page_size, head_dim], a
table gives each sequence's pages in order, pages lie in the pool in random order, and table entries past a sequence's last
page are -1.  Sequences that share a prefix name the same pages for it.
"""
import math
import random

import numpy as np
import torch

own = False

DEV = 'cuda'
TYPES = {'f32': torch.float32, 'f16': torch.float16, 'bf16': torch.bfloat16, 'e4m3': torch.float8_e4m3fn}
BYTES = {'f32': 4, 'f16': 2, 'bf16': 2, 'e4m3': 1}
THETA = 1e6
E4M3_MAX = 448.0


def listed():
    return [
        # the queries and keys of one decode step of 16 short requests on the 0.5B model: the smallest call
        _rotate('rotate_step_05b_f16', 16, 16, 64, 'f16', far=512),
        # a long prompt's chunk on the 7B model, positions past the trained length under YaRN scaling
        _rotate('rotate_prompt_7b_yarn_bf16', 2048, 32, 128, 'bf16', far=120000, yarn=4.0),
        # neighbouring pairs, the first 64 of 128 values of a head, 32-bit values, an odd number of rows
        _rotate('rotate_part_pairs_f32', 777, 12, 128, 'f32', rot=64, pairs=True, far=4096),
        # one decode step of 16 requests on the 1.5B model
        _append('append_step_15b_f16', 16, 'f16', 'f16', 12, 2, 128, 16, 2048),
        # a prefill chunk of three prompts on the 7B model
        _append('append_prompt_7b_bf16', 2048, 'bf16', 'bf16', 28, 4, 128, 64, 8192, seqs=3),
        # ragged prompts padded to one length (a fifth of the rows is padding) into a cache of 8 bits
        _append('append_rows_7b_e4m3', 777, 'bf16', 'e4m3', 28, 4, 128, 32, 4096, seqs=7, pad=0.2),
        # one token of a lone chat on the 0.5B model, nothing shared: latency counts
        _attend('attend_one_05b_f16', 'f16', 'f16', 14, 2, 64, 16, 1, 1, 0, 733, 733),
        # 16 requests of the 1.5B model under one system prompt, an ordinary decode step
        _attend('attend_step_15b_f16', 'f16', 'f16', 12, 2, 128, 16, 16, 1, 2048, 1, 512),
        # 32 requests of the 7B model about one document of 8192 tokens
        _attend('attend_step_7b_bf16', 'bf16', 'bf16', 28, 4, 128, 64, 32, 1, 8192, 64, 1024),
        # a large batch about two documents of 16384 tokens, cache of 8 bits
        _attend('attend_step_7b_e4m3', 'bf16', 'e4m3', 28, 4, 128, 128, 96, 2, 16384, 16, 2000),
        # 9 drafted tokens of each of 12 requests verified in one pass under a shared prefix of an odd length
        _attend('attend_draft_15b_f16', 'f16', 'f16', 12, 2, 128, 16, 12, 1, 1531, 16, 300, 9, 9),
        # the prompts of 8 requests on top of a shared prefix: the largest matrix work
        _attend('attend_prompts_7b_bf16', 'bf16', 'bf16', 28, 4, 128, 64, 8, 1, 4096, 100, 400, 100, 400),
    ]


def _rotate(name, rows, heads, hd, dtype, rot=None, pairs=False, far=4096, yarn=0.0):
    return {'name': name, 'kind': 'rotate', 'rows': rows, 'heads': heads, 'hd': hd, 'rot': rot or hd, 'pairs': pairs,
            'dtype': dtype, 'far': far, 'yarn': yarn}


def _append(name, rows, dtype, cache, nh, nkv, hd, page, far, seqs=0, pad=0.0, pairs=False, rot=None):
    """rows tokens of `seqs` sequences (0: one token each), cached positions below `far`, a share `pad` of padding rows."""
    return {'name': name, 'kind': 'append', 'rows': rows, 'dtype': dtype, 'cache': cache, 'nh': nh, 'nkv': nkv, 'hd': hd,
            'page': page, 'far': far, 'seqs': seqs, 'pad': pad, 'pairs': pairs, 'rot': rot or hd, 'yarn': 0.0}


def _attend(name, dtype, cache, nh, nkv, hd, page, batch, groups, shared, lo, hi, q_lo=1, q_hi=1):
    """batch sequences in `groups` groups, each group's sequences under `shared` common positions, lo..hi further
    positions of their own, of which the last q_lo..q_hi are the queries'."""
    return {'name': name, 'kind': 'attend', 'dtype': dtype, 'cache': cache, 'nh': nh, 'nkv': nkv, 'hd': hd, 'page': page,
            'batch': batch, 'groups': groups, 'shared': shared, 'lo': lo, 'hi': hi, 'q_lo': q_lo, 'q_hi': q_hi}


def draw(rng):
    """One more case of the same ranges."""
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(['rotate', 'append', 'attend', 'attend'])
    nh, nkv, hd = rng.choice([(14, 2, 64), (12, 2, 128), (28, 4, 128), (16, 16, 64), (8, 1, 128)])
    page = rng.choice([8, 16, 16, 24, 32, 64, 128])
    if kind == 'rotate':
        heads = rng.choice([nh + nkv, nh, nkv])
        dtype = rng.choice(['f32', 'f16', 'bf16'])
        c = _rotate(None, log(1, 1024 if dtype == 'f32' else 2048), heads, hd, dtype, rot=rng.choice([hd, hd, hd // 2]),
                    pairs=rng.random() < 0.4, far=log(64, 130000), yarn=rng.choice([0.0, 0.0, 2.0, 4.0]))
    elif kind == 'append':
        dtype = rng.choice(['f32', 'f16', 'bf16'])
        rows = log(1, 1024 if dtype == 'f32' else 2048)
        seqs = rng.choice([0, 0, rng.randint(1, 8)]) if rows <= 64 else rng.randint(1, 8)
        c = _append(None, rows, dtype, 'e4m3' if rng.random() < 0.3 else 'f16' if dtype == 'f32' else dtype, nh, nkv, hd, page,
                    max(2 * rows, log(256, 8192)), seqs=seqs, pad=rng.choice([0.0, 0.0, 0.2]), pairs=rng.random() < 0.3,
                    rot=rng.choice([hd, hd, hd // 2]))
    else:
        dtype = rng.choice(['f16', 'bf16'])
        cache = rng.choice([dtype, dtype, 'e4m3'])
        form = rng.choice(['step', 'step', 'step', 'draft', 'prompts'])
        if form == 'step':
            batch, q_lo, q_hi = log(1, 96), 1, 1
            shared, hi = rng.choice([0, log(64, 16384)]), log(16, min(4096, 80000 * 512 // (batch * nkv * hd)))
        elif form == 'draft':
            batch, q_hi = log(1, 16), rng.randint(2, 33)
            q_lo, shared, hi = rng.choice([q_hi, 1]), log(64, 4096), log(64, 1024)
        else:
            batch, q_hi = rng.randint(1, 8), log(40, 400)
            q_lo, shared, hi = max(1, q_hi // 4), log(64, 4096), q_hi
        lo = max(q_hi, hi // rng.choice([1, 4, 16]))
        hi = max(lo, hi)
        c = _attend(None, dtype, cache, nh, nkv, hd, page, batch, rng.randint(1, max(1, min(3, batch // 4))), shared, lo, hi,
                    q_lo, q_hi)
    c.pop('name', None)
    return c


# ------------------------------------------------------------------------------------------------ inputs from a seed
def _gen(seed, stream):
    return torch.Generator(device=DEV).manual_seed((seed * 1000003 + stream) % (2 ** 63))


def _frequencies(rot, yarn):
    """Angle per position of each pair (64 bits), and the factor on cosines and sines: plain, or YaRN with its usual
    parameters over an original length of 32768 positions."""
    inv = THETA ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    if not yarn:
        return inv, 1.0
    at = lambda turns: rot * math.log(32768 / (turns * 2 * math.pi)) / (2 * math.log(THETA))
    low, high = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), rot - 1)
    ramp = ((torch.arange(rot // 2, dtype=torch.float64) - low) / max(high - low, 1e-3)).clamp(0, 1)
    return inv / yarn * ramp + inv * (1 - ramp), 0.1 * math.log(yarn) + 1.0


def _scaling(yarn):
    return {'rope_type': 'yarn', 'factor': yarn, 'original_max_position_embeddings': 32768} if yarn else None


def _rotary(case):
    from seedplane_amd.paged import Rotary
    return Rotary(case['hd'], theta=THETA, rot_dim=case['rot'], layout='interleaved' if case['pairs'] else 'half',
                  scaling=_scaling(case['yarn']), device=DEV)


def _lay_out(rng, lens, shared, group_of, page):
    """A page table [sequences, most pages] over the fewest pages, in random order: the whole pages of a group's shared
    positions are common to its sequences; the rest of the sequence has pages of its own."""
    own_pages = [-(-n // page) - shared // page for n in lens]
    n_groups = group_of[-1] + 1
    total = n_groups * (shared // page) + sum(own_pages)
    order = rng.permutation(max(total, 1)).astype(np.int32)
    table = np.full((len(lens), max(1, max(shared // page + n for n in own_pages))), -1, dtype=np.int32)
    at = n_groups * (shared // page)
    for s, n in enumerate(own_pages):
        g = group_of[s]
        table[s, :shared // page] = order[g * (shared // page):(g + 1) * (shared // page)]
        table[s, shared // page:shared // page + n] = order[at:at + n]
        at += n
    return table, max(total, 1)


def _pool(g, shape, case, bias):
    """Pages whose values have the spread of a trained layer's keys or values: unit normal around a mean per channel."""
    x = torch.randn(shape, generator=g, device=DEV)
    x += bias * torch.randn((shape[1], 1, shape[3]), generator=g, device=DEV)
    if case['cache'] != 'e4m3':
        return x.to(TYPES[case['cache']]), None
    scale = (torch.rand(shape[1], generator=g, device=DEV) + 1.0) * (4.0 / E4M3_MAX)
    return (x / scale[:, None, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn), scale


def _int(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(DEV)


def prepare(case, seed):
    rng = np.random.default_rng([seed, 1])
    g = _gen(seed, 2)
    st = {'kind': case['kind'], 'case': case}
    if case['kind'] == 'rotate':
        # heads of a wider row, as the projection leaves queries, keys and values side by side
        wide = torch.randn((case['rows'], case['heads'] + 4, case['hd']), generator=g, device=DEV).to(TYPES[case['dtype']])
        st['x'] = wide[:, :case['heads']]
        st['pos'] = _int(rng.integers(0, case['far'], case['rows']))
    elif case['kind'] == 'append':
        _prepare_append(case, st, rng, g)
    else:
        _prepare_attend(case, st, rng, g)
    if case['kind'] != 'attend':
        inv, factor = _frequencies(case['rot'], case['yarn'])
        st['inv'], st['factor'] = inv.to(DEV), factor
    if own:
        if case['kind'] != 'attend':
            st['rotary'] = _rotary(case)
        if case['kind'] != 'rotate':
            from seedplane_amd.paged import PagedKV
            st['kv'] = PagedKV(st['k'], st['v'], k_scale=st['k_scale'], v_scale=st['v_scale'])
        if case['kind'] == 'attend':
            from seedplane_amd.paged import AttentionPlan
            st['plan'] = AttentionPlan(case['nh'], case['nkv'], case['hd'], max_rows=sum(st['q_lens']), max_seqs=case['batch'],
                                       device=DEV)
            st['plan'].set(st['q_lens'], st['kv_lens'], st['sharing'])
    return st


def _lengths(case):
    """The lengths of a case, the same for every seed (the shapes of the inputs do not depend on it).  append: the new rows
    of each sequence and the position of its first; attend: the query rows of each sequence and its cached positions, those of
    the queries included."""
    r = random.Random(repr(sorted((k, v) for k, v in case.items() if k != 'name')))
    if case['kind'] == 'append':
        counts = [1] * case['rows']
        if case['seqs']:
            live = case['rows'] - int(case['rows'] * case['pad'])
            cuts = [0, *sorted(r.randint(0, live) for _ in range(case['seqs'] - 1)), live]
            counts = [b - a for a, b in zip(cuts, cuts[1:])]
        return counts, [r.randint(0, case['far'] - n) for n in counts]
    q_lens = [r.randint(case['q_lo'], case['q_hi']) for _ in range(case['batch'])]
    if case['q_hi'] > 33:                                    # prompts: everything after the prefix is new
        return q_lens, [case['shared'] + q for q in q_lens]
    return q_lens, [case['shared'] + max(q, r.randint(case['lo'], case['hi'])) for q in q_lens]


def _prepare_append(case, st, rng, g):
    rows, page, nh, nkv, hd = case['rows'], case['page'], case['nh'], case['nkv'], case['hd']
    counts, starts = _lengths(case)
    n_seq, live = len(counts), sum(counts)
    seq = np.concatenate([np.full(n, s) for s, n in enumerate(counts)] + [np.full(rows - live, -1)])
    pos = np.concatenate([np.arange(a, a + n) for a, n in zip(starts, counts)] + [np.zeros(rows - live)])
    lens = [a + n for a, n in zip(starts, counts)]
    # the pool holds the pages that are written and a few more; earlier pages are elsewhere (their entries stay -1)
    table = np.full((n_seq, -(-case['far'] // page)), -1, dtype=np.int32)
    spans = [(a // page, -(-b // page)) for a, b in zip(starts, lens)]
    total = rows // page + 2 * n_seq + 3
    order, at = rng.permutation(total), 0
    for s, (a, b) in enumerate(spans):
        table[s, a:b] = order[at:at + b - a]
        at += b - a
    st['seq'], st['pos'], st['table'] = _int(seq), _int(pos), _int(table)
    qkv = torch.randn((rows, (nh + 2 * nkv) * hd), generator=g, device=DEV).to(TYPES[case['dtype']])
    heads = qkv.view(rows, nh + 2 * nkv, hd)
    st['q'], st['kn'], st['vn'] = heads[:, :nh], heads[:, nh:nh + nkv], heads[:, nh + nkv:]
    st['q_out'] = torch.zeros((rows, nh, hd), dtype=heads.dtype, device=DEV)
    shape = (total, nkv, page, hd)
    st['k'], st['k_scale'] = _pool(g, shape, case, 0.0)
    st['v'], st['v_scale'] = _pool(g, shape, case, 0.0)


def _prepare_attend(case, st, rng, g):
    B, page, nh, nkv, hd, shared = case['batch'], case['page'], case['nh'], case['nkv'], case['hd'], case['shared']
    q_lens, kv_lens = _lengths(case)
    group_of = sorted(i % case['groups'] for i in range(B))
    table, total = _lay_out(rng, kv_lens, shared, group_of, page)
    whole = shared // page * page                            # the positions whose pages are common
    st['q_lens'], st['kv_lens'] = q_lens, kv_lens
    st['sharing'] = [(group_of.count(i), whole) for i in range(case['groups'])]
    st['table'] = _int(table)
    st['row_seq'] = _int(np.repeat(np.arange(B), q_lens))
    st['row_idx'] = _int(np.concatenate([np.arange(n) for n in q_lens]))
    st['row_pos'] = _int(np.concatenate([np.arange(n - q, n) for q, n in zip(q_lens, kv_lens)]))
    st['most_q'], st['most_kv'] = max(q_lens), max(kv_lens)
    shape = (total, nkv, page, hd)
    st['k'], st['k_scale'] = _pool(g, shape, case, 0.5)
    st['v'], st['v_scale'] = _pool(g, shape, case, 0.0)
    st['q'] = (torch.randn((sum(q_lens), nh, hd), generator=g, device=DEV) * 1.5).to(TYPES[case['dtype']])


# ------------------------------------------------------------------------------------------------ run
def run(st):
    case = st['case']
    if st['kind'] == 'rotate':
        if own:
            return st['rotary'].apply(st['x'], st['pos'])
        return _turned(st['x'].float(), st).to(st['x'].dtype)
    if st['kind'] == 'append':
        if own:
            st['kv'].append(st['kn'], st['vn'], st['seq'], st['pos'], st['table'], rotary=st['rotary'], q=st['q'],
                            q_out=st['q_out'])
        else:
            _append_plain(st, case)
        return {'q': st['q_out'], 'k': st['k'], 'v': st['v']}
    if own:
        return st['plan'].run(st['q'], st['kv'], st['table'])
    return _attend_plain(st, case)


def _turned(x, st):
    """x [rows, heads, head_dim] in 32 bits, the first `rot` values of each head rotated; angles of far positions in 64."""
    rot, pairs = st['case']['rot'], st['case']['pairs']
    angle = st['pos'].double()[:, None] * st['inv']
    c = (angle.cos() * st['factor']).float()[:, None, :]
    s = (angle.sin() * st['factor']).float()[:, None, :]
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if pairs else (x[..., :rot // 2], x[..., rot // 2:rot])
    first, second = a * c - b * s, b * c + a * s
    y = torch.stack([first, second], dim=-1).flatten(-2) if pairs else torch.cat([first, second], dim=-1)
    return torch.cat([y, x[..., rot:]], dim=-1)


def _append_plain(st, case):
    nh, page = case['nh'], case['page']
    turned = _turned(torch.cat([st['q'], st['kn']], dim=1).float(), st)
    live = st['seq'] >= 0
    st['q_out'].copy_(torch.where(live[:, None, None], turned[:, :nh].to(st['q_out'].dtype), st['q_out']))
    row = live.nonzero()[:, 0]
    pos = st['pos'][row].long()
    where = st['table'][st['seq'][row].long(), pos // page].long()
    for name, value, scale in (('k', turned[:, nh:], st['k_scale']), ('v', st['vn'].float(), st['v_scale'])):
        value = value[row]
        if scale is not None:
            value = (value / scale[:, None]).clamp(-E4M3_MAX, E4M3_MAX)
        pool = st[name].view(torch.uint8) if scale is not None else st[name]
        value = value.to(st[name].dtype)
        pool[where, :, pos % page] = value.view(torch.uint8) if scale is not None else value


def _attend_plain(st, case):
    """Every sequence's keys and values gathered to the longest length, scores with a mask, softmax, weighted sum."""
    B, nh, nkv, hd, page = case['batch'], case['nh'], case['nkv'], case['hd'], case['page']
    Q, L = st['most_q'], st['most_kv']
    at = torch.arange(L, device=DEV)
    pages = st['table'][:, at // page].clamp_min(0).long()                        # [B, L]
    off = (at % page).expand(B, L)

    def gathered(pool, scale):
        x = pool.view(torch.uint8) if scale is not None else pool
        x = x[pages, :, off]                                                       # [B, L, nkv, hd]
        x = x.view(pool.dtype).float() if scale is not None else x.float()
        return x * scale[:, None] if scale is not None else x
    k = gathered(st['k'], st['k_scale']).permute(0, 2, 3, 1).contiguous()          # [B, nkv, hd, L]
    seq, idx = st['row_seq'].long(), st['row_idx'].long()
    q = torch.zeros((B, Q, nh, hd), device=DEV)
    q[seq, idx] = st['q'].float()
    last = torch.full((B, Q), -1, device=DEV, dtype=torch.int32)
    last[seq, idx] = st['row_pos']
    q = q.view(B, Q, nkv, nh // nkv, hd).permute(0, 2, 1, 3, 4).reshape(B, nkv, Q * (nh // nkv), hd)
    s = torch.matmul(q, k) * (1.0 / math.sqrt(hd))
    del k
    s = s.view(B, nkv, Q, nh // nkv, L).masked_fill(at > last[:, None, :, None, None], -torch.inf)
    m = s.amax(-1, keepdim=True)
    e = (s - torch.where(m == -torch.inf, torch.zeros_like(m), m)).exp()
    del s
    den = e.sum(-1, keepdim=True)
    v = gathered(st['v'], st['v_scale']).permute(0, 2, 1, 3).contiguous()          # [B, nkv, L, hd]
    o = torch.matmul(e.view(B, nkv, Q * (nh // nkv), L), v).view(B, nkv, Q, nh // nkv, hd) / den.clamp_min(1e-30)
    return o.permute(0, 2, 1, 3, 4).reshape(B, Q, nh, hd)[seq, idx].to(st['q'].dtype)


# ------------------------------------------------------------------------------------------------ what a pass needs
def work(case):
    if case['kind'] == 'rotate':
        n = case['rows'] * case['heads']
        return {'bytes': 2 * n * case['hd'] * BYTES[case['dtype']] + 4 * case['rows'], 'flops': 3 * n * case['rot']}
    if case['kind'] == 'append':
        rows = sum(_lengths(case)[0])
        q, kv, b = case['nh'] * case['hd'], 2 * case['nkv'] * case['hd'], BYTES[case['dtype']]
        return {'bytes': rows * (2 * q * b + kv * (b + BYTES[case['cache']])) + 12 * case['rows'],
                'flops': 3 * rows * (case['nh'] + case['nkv']) * case['rot']}
    q_lens, kv_lens = _lengths(case)
    whole = case['shared'] // case['page'] * case['page']
    read = case['groups'] * whole + sum(n - whole for n in kv_lens)
    pairs = sum(q * n - q * (q - 1) // 2 for q, n in zip(q_lens, kv_lens))
    return {'bytes': 2 * read * case['nkv'] * case['hd'] * BYTES[case['cache']] +
            2 * sum(q_lens) * case['nh'] * case['hd'] * BYTES[case['dtype']],
            'flops': 4 * pairs * case['nh'] * case['hd']}


# ------------------------------------------------------------------------------------------------ 64-bit results
def _turn_exact(x, pos, case):
    """Rotation as a complex product, from its own statement of the frequencies."""
    rot = case['rot']
    j = np.arange(rot // 2)
    inv, factor = np.exp(-np.log(THETA) * 2 * j / rot), 1.0
    if case['yarn']:
        # a pair that turns over 32 times within the original length keeps its frequency, one that turns less than once is
        # slowed by the factor; between them, linearly in the pair's index (the borders rounded outwards)
        edge = [rot * np.log(32768.0 / (2 * np.pi * t)) / (2 * np.log(THETA)) for t in (32.0, 1.0)]
        lo, hi = max(0, int(np.floor(edge[0]))), min(rot - 1, int(np.ceil(edge[1])))
        keep = 1.0 - np.clip((j - lo) / max(hi - lo, 1e-3), 0.0, 1.0)
        inv = inv * (keep + (1.0 - keep) / case['yarn'])
        factor = 1.0 + 0.1 * np.log(case['yarn'])
    turn = factor * np.exp(1j * pos.cpu().numpy().astype(np.float64)[:, None] * inv)
    turn = torch.from_numpy(turn).to(DEV)[:, None, :]
    y = x.double().clone()
    first, second = (slice(0, rot, 2), slice(1, rot, 2)) if case['pairs'] else (slice(0, rot // 2), slice(rot // 2, rot))
    z = torch.complex(y[..., first], y[..., second]) * turn
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _e4m3_exact(x):
    """The nearest value with 3 fraction bits, exponents from -6, at most 448; ties to even."""
    x = x.clamp(-E4M3_MAX, E4M3_MAX)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def exact(case, seed):
    st = prepare(case, seed)
    if case['kind'] == 'rotate':
        return _turn_exact(st['x'], st['pos'], case)
    if case['kind'] == 'append':
        q, k, v = st['q_out'].double(), st['k'].double(), st['v'].double()
        seq, pos, table = st['seq'].tolist(), st['pos'].tolist(), st['table'].tolist()
        rq, rk = _turn_exact(st['q'], st['pos'], case), _turn_exact(st['kn'], st['pos'], case)
        for pool, new, scale in ((k, rk, st['k_scale']), (v, st['vn'].double(), st['v_scale'])):
            if scale is not None:
                new = _e4m3_exact(new / scale.double()[:, None])
            for i, s in enumerate(seq):
                if s >= 0:
                    pool[table[s][pos[i] // case['page']], :, pos[i] % case['page']] = new[i]
        alive = torch.tensor([i for i, s in enumerate(seq) if s >= 0], device=DEV, dtype=torch.long)
        q[alive] = rq[alive]
        return {'q': q, 'k': k, 'v': v}
    nh, nkv, hd, page = case['nh'], case['nkv'], case['hd'], case['page']
    out, r0 = torch.zeros((sum(st['q_lens']), nh, hd), dtype=torch.float64, device=DEV), 0
    for s, (nq, n) in enumerate(zip(st['q_lens'], st['kv_lens'])):
        pages = st['table'][s, :-(-n // page)].long()
        rows = []
        for pool, scale in ((st['k'], st['k_scale']), (st['v'], st['v_scale'])):
            x = pool.view(torch.uint8)[pages].view(pool.dtype).double() if scale is not None else pool[pages].double()
            x = x if scale is None else x * scale.double()[:, None, None]
            rows.append(x.permute(1, 0, 2, 3).reshape(nkv, -1, hd)[:, :n])
        hidden = torch.arange(n, device=DEV)[None, :] > torch.arange(n - nq, n, device=DEV)[:, None]
        for h in range(nh):
            kv = h // (nh // nkv)
            w = st['q'][r0:r0 + nq, h].double() @ rows[0][kv].T.contiguous() / hd ** 0.5
            w = torch.softmax(w.masked_fill(hidden, -torch.inf), dim=-1)
            out[r0:r0 + nq, h] = w @ rows[1][kv].contiguous()
        r0 += nq
    return out
