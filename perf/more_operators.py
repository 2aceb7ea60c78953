"""Operators of a server that searches with beams over a paged K/V cache of 8 bits, as cases that can be timed and checked one by
one: appending to pages whose codes have a scale for each block of positions and head, and reading positions back (`append`);
attention over such pages (`attend`); the selection of the next beams (`beam`); sequences that continue others' pages (`fork`);
sequences that end, pages that close up and sequences that begin (`turnover`).

Head shapes are those of the Qwen2-0.5B / 1.5B / 7B presets (14/2 heads of 64, 12/2 of 128, 28/4 of 128), the vocabulary is theirs
(151936), except where a case says otherwise.  Pools are [pages, kv_heads, page_size, head_dim], scales [pages, kv_heads, blocks of
a page]; a table gives each sequence's pages in order, -1 behind the last.
"""
import math
import random

import numpy as np
import torch

own = False

DEV = 'cuda'
TYPES = {'f32': torch.float32, 'f16': torch.float16, 'bf16': torch.bfloat16, 'int8': torch.int8, 'e4m3': torch.float8_e4m3fn}
BYTES = {'f32': 4, 'f16': 2, 'bf16': 2, 'int8': 1, 'e4m3': 1}
MOST = {'int8': 127.0, 'e4m3': 448.0}
LEAST_SCALE = 2.0 ** -60
THETA = 1e6
VOCAB = 151936


def listed():
    return [
        # one decode step of 16 requests on the 1.5B model: most blocks are continued
        _append('append_step_15b_int8', 16, 'f16', 'int8', 12, 2, 128, 16, 16, 2048),
        # a prefill chunk of five prompts on the 7B model, a tenth of the rows padding
        _append('append_prompt_7b_int8', 1777, 'bf16', 'int8', 28, 4, 128, 64, 32, 6000, seqs=5, pad=0.1),
        # one token of a lone chat on the 0.5B model: latency counts
        _attend('attend_one_05b_int8', 'f16', 'int8', 14, 2, 64, 16, 16, 1, 1, 0, 1201, 1201),
        # 48 requests of the 7B model under one system prompt, an ordinary decode step
        _attend('attend_step_7b_e4m3', 'bf16', 'e4m3', 28, 4, 128, 64, 16, 48, 1, 4096, 64, 2000),
        # 8 long conversations on the 7B model, nothing shared
        _attend('attend_long_7b_int8', 'bf16', 'int8', 28, 4, 128, 128, 64, 8, 1, 0, 20000, 40000),
        # the prompts of 6 requests on top of a shared prefix on the 1.5B model
        _attend('attend_prompts_15b_int8', 'f16', 'int8', 12, 2, 128, 32, 32, 6, 1, 1000, 300, 900, 300, 900),
        # one request with 4 beams, fp32 logits as the engine gives them
        _beam('beam_one_f32', 1, 4, VOCAB, 'f32'),
        # 32 requests with 8 beams each
        _beam('beam_batch_bf16', 32, 8, VOCAB, 'bf16'),
        # 4 beams of one request on the 1.5B model's 28 layers, fp16 cache
        _pages('fork_one_15b_f16', 'fork', 28, 1, 4, 'f16', 2, 128, 16, 16, 300, 600),
        # 16 requests with 8 beams each on the 7B model's 28 layers, cache of 8 bits
        _pages('fork_batch_7b_int8', 'fork', 28, 16, 8, 'int8', 4, 128, 64, 16, 500, 1500),
        # 16 short requests of the 0.5B model's 24 layers, half of them replaced
        _pages('turnover_05b_f16', 'turnover', 24, 16, 1, 'f16', 2, 64, 16, 16, 20, 200),
        # 64 requests of 16 layers of the 7B model, half of them replaced
        _pages('turnover_7b_bf16', 'turnover', 16, 64, 1, 'bf16', 4, 128, 64, 16, 200, 2500),
    ]


def _append(name, rows, dtype, cache, nh, nkv, hd, page, block, far, seqs=0, pad=0.0, pairs=False, rot=None):
    """rows tokens of `seqs` sequences (0: one token each), positions below `far`, a share `pad` of padding rows."""
    return {'name': name, 'kind': 'append', 'rows': rows, 'dtype': dtype, 'cache': cache, 'nh': nh, 'nkv': nkv, 'hd': hd,
            'page': page, 'block': block, 'far': far, 'seqs': seqs, 'pad': pad, 'pairs': pairs, 'rot': rot or hd}


def _attend(name, dtype, cache, nh, nkv, hd, page, block, batch, groups, shared, lo, hi, q_lo=1, q_hi=1):
    """batch sequences in `groups` groups, each under `shared` common positions, lo..hi further ones of their own, of which the
    last q_lo..q_hi are the queries'."""
    return {'name': name, 'kind': 'attend', 'dtype': dtype, 'cache': cache, 'nh': nh, 'nkv': nkv, 'hd': hd, 'page': page,
            'block': block, 'batch': batch, 'groups': groups, 'shared': shared, 'lo': lo, 'hi': hi, 'q_lo': q_lo, 'q_hi': q_hi}


def _beam(name, batch, beams, vocab, dtype, first=False, masked=0.0):
    """first: only one beam of each request lives; masked: the share of the vocabulary that a grammar forbids."""
    return {'name': name, 'kind': 'beam', 'batch': batch, 'beams': beams, 'vocab': vocab, 'dtype': dtype, 'first': first,
            'masked': masked}


def _pages(name, kind, layers, batch, beams, cache, nkv, hd, page, block, lo, hi):
    """batch requests of lo..hi positions, each with `beams` sequences whose last eighth is their own."""
    return {'name': name, 'kind': kind, 'layers': layers, 'batch': batch, 'beams': beams, 'cache': cache, 'nkv': nkv, 'hd': hd,
            'page': page, 'block': block, 'lo': lo, 'hi': hi}


def draw(rng):
    """One more case of the same ranges."""
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(['append', 'attend', 'attend', 'beam', 'fork', 'turnover'])
    nh, nkv, hd = rng.choice([(14, 2, 64), (12, 2, 128), (28, 4, 128), (16, 16, 64), (8, 1, 128)])
    page, block = rng.choice([(16, 16), (32, 16), (32, 32), (48, 16), (64, 16), (64, 32), (64, 64), (128, 64), (128, 128)])
    cache = rng.choice(['int8', 'int8', 'e4m3'])
    if kind == 'append':
        rows = log(1, 1777)
        seqs = rng.choice([0, 0, rng.randint(1, 8)]) if rows <= 64 else rng.randint(1, 8)
        c = _append(None, rows, rng.choice(['f32', 'f16', 'bf16']), cache, nh, nkv, hd, page, block, max(2 * rows, log(256, 8192)),
                    seqs=seqs, pad=rng.choice([0.0, 0.0, 0.2]), pairs=rng.random() < 0.3, rot=rng.choice([hd, hd, hd // 2]))
    elif kind == 'attend':
        form = rng.choice(['step', 'step', 'long', 'draft', 'prompts'])
        q_lo = q_hi = 1
        if form == 'step':
            batch, shared = log(1, 64), rng.choice([0, log(64, 8192)])
            hi = log(16, min(3000, 80000 * 512 // (batch * nkv * hd)))
        elif form == 'long':
            batch, shared, hi = rng.randint(1, 8), 0, log(4000, 40000 if nkv < 16 else 16000)
        elif form == 'draft':
            batch, q_hi = log(1, 16), rng.randint(2, 33)
            q_lo, shared, hi = rng.choice([q_hi, 1]), log(64, 4096), log(64, 1024)
        else:
            batch, q_hi = rng.randint(1, 6), log(40, 900)
            q_lo, shared, hi = max(1, q_hi // 4), log(64, 1000), q_hi
        lo = max(q_hi, hi // rng.choice([1, 4, 16]))
        c = _attend(None, rng.choice(['f16', 'bf16']), cache, nh, nkv, hd, page, block, batch, rng.randint(1, max(1, min(3, batch // 4))),
                    shared, lo, max(lo, hi), q_lo, q_hi)
    elif kind == 'beam':
        c = _beam(None, log(1, 32), rng.randint(1, 8), rng.choice([VOCAB, VOCAB, log(1000, VOCAB)]), rng.choice(['f32', 'f16', 'bf16']),
                  first=rng.random() < 0.2, masked=rng.choice([0.0, 0.0, 0.5, 0.999]))
        if c['batch'] * c['beams'] * c['vocab'] * BYTES[c['dtype']] > 32 * 8 * VOCAB * 2:
            c['dtype'] = 'bf16'
    else:
        turnover = kind == 'turnover'
        cache = rng.choice([cache, 'f16', 'bf16'])
        layers, hi = rng.randint(1, 28), log(40, 2000)
        batch, beams = (log(2, 64), 1) if turnover else (log(1, 16), rng.randint(2, 8))
        page, block = rng.choice([(16, 16), (32, 16), (64, 16), (64, 64)])
        layers = max(1, min(layers, 16 * 64 * 1300 * 512 * 2 // (batch * beams * hi * nkv * hd * BYTES[cache])))
        c = _pages(None, kind, layers, batch, beams, cache, nkv, hd, page, block, max(1, hi // rng.choice([1, 4, 16])), hi)
    c.pop('name', None)
    return c


# ------------------------------------------------------------------------------------------------ inputs from a seed
def _gen(seed, stream):
    return torch.Generator(device=DEV).manual_seed((seed * 1000003 + stream) % (2 ** 63))


def _int(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(DEV)


def _fixed(case):
    """Lengths are the same for every seed (the shapes of inputs and outputs do not depend on it)."""
    return random.Random(repr(sorted((k, v) for k, v in case.items() if k != 'name')))


def _codes(x, cache, block):
    """Values [.., page, hd] as codes and scales [.., page / block], each block at the full range of the codes."""
    b = x.unflatten(-2, (-1, block))
    scale = b.abs().amax((-2, -1)) / MOST[cache]
    b = b / scale[..., None, None]
    return (b.round().to(torch.int8) if cache == 'int8' else b.to(torch.float8_e4m3fn)).flatten(-3, -2), scale


def _values(codes, scale, block):
    """Codes [.., page, hd] with scales [.., page / block] as fp32 values."""
    return (codes.float().unflatten(-2, (-1, block)) * scale[..., None, None]).flatten(-3, -2)


def _pool(g, shape, case, bias):
    """Pages whose values have the spread of a trained layer's keys or values: unit normal around a mean per channel, some
    positions larger than others."""
    x = torch.randn(shape, generator=g, device=DEV)
    x += bias * torch.randn((shape[1], 1, shape[3]), generator=g, device=DEV)
    x *= 0.5 + torch.rand((*shape[:3], 1), generator=g, device=DEV)
    return _codes(x, case['cache'], case['block'])


def prepare(case, seed):
    rng = np.random.default_rng([seed, 1])
    st = {'kind': case['kind'], 'case': case}
    {'append': _prepare_append, 'attend': _prepare_attend, 'beam': _prepare_beam, 'fork': _prepare_pages,
     'turnover': _prepare_pages}[case['kind']](case, st, rng, _gen(seed, 2))
    return st


def _append_lengths(case):
    """The new rows of each sequence and the position of its first."""
    r = _fixed(case)
    counts = [1] * case['rows']
    if case['seqs']:
        live = case['rows'] - int(case['rows'] * case['pad'])
        cuts = [0, *sorted(r.randint(0, live) for _ in range(case['seqs'] - 1)), live]
        counts = [b - a for a, b in zip(cuts, cuts[1:])]
    return counts, [r.randint(0, case['far'] - n) for n in counts]


def _prepare_append(case, st, rng, g):
    rows, page, block, nh, nkv, hd = (case[k] for k in ('rows', 'page', 'block', 'nh', 'nkv', 'hd'))
    counts, starts = _append_lengths(case)
    n_seq, live = len(counts), sum(counts)
    st['seq'] = _int(np.concatenate([np.full(n, s) for s, n in enumerate(counts)] + [np.full(rows - live, -1)]))
    st['pos'] = _int(np.concatenate([np.arange(a, a + n) for a, n in zip(starts, counts)] + [np.zeros(rows - live)]))
    # the pool holds the pages that are written and a few more; earlier pages are elsewhere (their entries stay -1)
    table = np.full((n_seq, -(-case['far'] // page)), -1, dtype=np.int32)
    spans = [(a // page, -(-(a + n) // page)) for a, n in zip(starts, counts)]
    total = rows // page + 2 * n_seq + 3
    order, at = rng.permutation(total), 0
    for s, (a, b) in enumerate(spans):
        if counts[s]:
            table[s, a:b] = order[at:at + b - a]
            at += b - a
    st['table'] = _int(table)
    # what is read back: every block that the call writes, from its first position to the last new one
    held = [(s, p) for s, (a, n) in enumerate(zip(starts, counts)) if n for p in range(a // block * block, a + n)]
    st['read_seq'], st['read_pos'] = _int([s for s, _ in held]), _int([p for _, p in held])
    heads = torch.randn((rows, nh + 2 * nkv, hd), generator=g, device=DEV).to(TYPES[case['dtype']])
    st['q'], st['kn'], st['vn'] = heads[:, :nh], heads[:, nh:nh + nkv], heads[:, nh + nkv:]
    st['q_out'] = torch.zeros((rows, nh, hd), dtype=heads.dtype, device=DEV)
    shape = (total, nkv, page, hd)
    (st['k'], st['ks']), (st['v'], st['vs']) = (_pool(g, shape, case, 0.0) for _ in range(2))
    st['inv'] = (THETA ** (-torch.arange(0, case['rot'], 2, dtype=torch.float64) / case['rot'])).to(DEV)
    if own:
        from seedplane_amd.paged import PagedKV, Rotary
        st['kv'] = PagedKV(st['k'], st['v'], k_scale=st['ks'], v_scale=st['vs'])
        st['rotary'] = Rotary(hd, theta=THETA, rot_dim=case['rot'], layout='interleaved' if case['pairs'] else 'half', device=DEV)


def _attend_lengths(case):
    """The query rows of each sequence and its cached positions, those of the queries included."""
    r = _fixed(case)
    q_lens = [r.randint(case['q_lo'], case['q_hi']) for _ in range(case['batch'])]
    if case['q_hi'] > 33:                                    # prompts: everything after the prefix is new
        return q_lens, [case['shared'] + q for q in q_lens]
    return q_lens, [case['shared'] + max(q, r.randint(case['lo'], case['hi'])) for q in q_lens]


def _lay_out(rng, lens, shared, group_of, page):
    """A page table over the fewest pages, in random order: the whole pages of a group's shared positions are common to its
    sequences; the rest of the sequence has pages of its own."""
    own_pages = [-(-n // page) - shared // page for n in lens]
    n_groups = group_of[-1] + 1
    total = n_groups * (shared // page) + sum(own_pages)
    order = rng.permutation(max(total, 1)).astype(np.int32)
    table = np.full((len(lens), max(1, max(shared // page + n for n in own_pages))), -1, dtype=np.int32)
    at = n_groups * (shared // page)
    for s, n in enumerate(own_pages):
        i = group_of[s]
        table[s, :shared // page] = order[i * (shared // page):(i + 1) * (shared // page)]
        table[s, shared // page:shared // page + n] = order[at:at + n]
        at += n
    return table, max(total, 1)


def _prepare_attend(case, st, rng, g):
    B, page, nh, nkv, hd, shared = (case[k] for k in ('batch', 'page', 'nh', 'nkv', 'hd', 'shared'))
    q_lens, kv_lens = _attend_lengths(case)
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
    (st['k'], st['ks']), (st['v'], st['vs']) = (_pool(g, shape, case, bias) for bias in (0.5, 0.0))
    st['q'] = (torch.randn((sum(q_lens), nh, hd), generator=g, device=DEV) * 1.5).to(TYPES[case['dtype']])
    if own:
        from seedplane_amd.paged import AttentionPlan, PagedKV
        st['kv'] = PagedKV(st['k'], st['v'], k_scale=st['ks'], v_scale=st['vs'])
        st['plan'] = AttentionPlan(nh, nkv, hd, max_rows=sum(q_lens), max_seqs=B, device=DEV)
        st['plan'].set(q_lens, kv_lens, st['sharing'])


def _prepare_beam(case, st, rng, g):
    B, K, V = case['batch'], case['beams'], case['vocab']
    # logits of a trained model: a wide body and a few likely tokens
    x = torch.randn((B * K, V), generator=g, device=DEV) * 2.5
    top = torch.randint(0, V, (B * K, 20), generator=g, device=DEV)
    x.scatter_add_(1, top, torch.rand((B * K, 20), generator=g, device=DEV) * 12)
    if case['masked']:
        forbidden = torch.rand(V, generator=g, device=DEV) < case['masked']
        forbidden[:50] = False
        x[:, forbidden] = -torch.inf
    st['logits'] = x.to(TYPES[case['dtype']])
    st['scores'] = -torch.rand((B, K), generator=g, device=DEV) * 3 - 20
    if case['first']:
        st['scores'][:, 0] = 0
        st['scores'][:, 1:] = -torch.inf
    st['eos'] = int(top[0, 0])


def _page_lengths(case):
    """The positions of each request, and those at its start that its beams share."""
    r = _fixed(case)
    lens = [r.randint(case['lo'], case['hi']) for _ in range(case['batch'])]
    if case['beams'] == 1:
        return lens, [0] * len(lens)
    return lens, [n * 7 // 8 // case['page'] * case['page'] for n in lens]


def _prepare_pages(case, st, rng, g):
    page, K, layers, nkv, hd = (case[k] for k in ('page', 'beams', 'layers', 'nkv', 'hd'))
    lens, common = _page_lengths(case)
    S, width = len(lens) * K, -(-max(lens) // page) + 1
    used = sum(c // page + K * (-(-n // page) - c // page) for n, c in zip(lens, common))
    total = used + S + 3
    order, at = np.arange(total), 0
    if K > 1:                                                # beams that have forked before: pages lie anywhere
        order = rng.permutation(total)
    table = np.full((S, width), -1, dtype=np.int32)
    for b, (n, c) in enumerate(zip(lens, common)):
        first, more = order[at:at + c // page], -(-n // page) - c // page
        at += c // page
        for k in range(K):
            table[b * K + k, :c // page] = first
            table[b * K + k, c // page:c // page + more] = order[at:at + more]
            at += more
    st['table'], st['lengths'] = _int(table), _int(np.repeat(lens, K))
    st['holders'] = _int(np.bincount(table[table >= 0], minlength=total))
    st['missing'] = torch.zeros(1, dtype=torch.int32, device=DEV)
    shape = (layers, 2, total, nkv, page, hd)
    if case['cache'] in MOST:
        codes = torch.randint(-127, 128, shape, generator=g, device=DEV, dtype=torch.int8)
        st['pool'] = codes if case['cache'] == 'int8' else codes.abs().clamp(max=110).view(torch.float8_e4m3fn)
        st['scale'] = torch.rand((layers, 2, total, nkv, page // case['block']), generator=g, device=DEV)
    else:
        st['pool'] = torch.randn(shape, generator=g, device=DEV, dtype=TYPES[case['cache']])
        st['scale'] = None
    if case['kind'] == 'fork':
        # each beam continues one of its request's beams, the better ones more often
        likely = rng.integers(0, K, (len(lens), K)) * rng.random((len(lens), K))
        st['parents'] = _int((np.arange(len(lens))[:, None] * K + np.sort(likely.astype(int), axis=1)).reshape(-1))
    else:
        halves = [np.arange(S)[i::2] for i in range(2)]
        st['ends'] = [_int(h) for h in halves]
        st['begins'] = [_int(np.where(np.isin(np.arange(S), h), lens, 0)) for h in halves]
        st['turn'] = 0
    if own:
        from seedplane_amd.paged import PagedKV
        from seedplane_amd.pages import PagePool
        caches = [PagedKV(st['pool'][i, 0], st['pool'][i, 1], *(() if st['scale'] is None else (st['scale'][i, 0], st['scale'][i, 1])))
                  for i in range(layers)]
        st['pages'] = PagePool(caches, S, width)
        for name in ('table', 'lengths', 'holders'):
            getattr(st['pages'], name).copy_(st[name])
            st[name] = getattr(st['pages'], name)
        st['missing'] = st['pages'].missing


# ------------------------------------------------------------------------------------------------ run
def run(st):
    case = st['case']
    if st['kind'] == 'append':
        dtype = st['q'].dtype if st['q'].dtype != torch.float32 else torch.float16
        if own:
            st['kv'].append(st['kn'], st['vn'], st['seq'], st['pos'], st['table'], rotary=st['rotary'], q=st['q'],
                            q_out=st['q_out'])
            k, v = st['kv'].read(st['read_seq'], st['read_pos'], st['table'], dtype=dtype)
        else:
            _append_plain(st, case)
            k, v = _read_plain(st, case, dtype)
        return {'q': st['q_out'], 'k': k, 'v': v, 'ks': st['ks'], 'vs': st['vs']}
    if st['kind'] == 'attend':
        return st['plan'].run(st['q'], st['kv'], st['table']) if own else _attend_plain(st, case)
    if st['kind'] == 'beam':
        if own:
            from seedplane_amd.beam import beam_select
            return tuple(beam_select(st['logits'], st['scores'], eos=st['eos']))
        return _beam_plain(st, case)
    if st['kind'] == 'fork':
        if own:
            st['pages'].fork(st['parents'])
        else:
            _fork_plain(st, case)
    else:
        ends, begins = st['ends'][st['turn']], st['begins'][st['turn']]
        st['turn'] ^= 1
        if own:
            st['pages'].free(ends)
            st['pages'].compact()
            st['pages'].grow(begins)
        else:
            _free_plain(st, ends)
            _compact_plain(st)
            _grow_plain(st, case, begins)
    return {k: st[k] for k in ('table', 'lengths', 'holders', 'missing', 'pool', 'scale')}


def _turned(x, st):
    """x [rows, heads, head_dim] in 32 bits, the first `rot` values of each head rotated; angles of far positions in 64."""
    rot, pairs = st['case']['rot'], st['case']['pairs']
    angle = st['pos'].double()[:, None] * st['inv']
    c, s = angle.cos().float()[:, None, :], angle.sin().float()[:, None, :]
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if pairs else (x[..., :rot // 2], x[..., rot // 2:rot])
    first, second = a * c - b * s, b * c + a * s
    y = torch.stack([first, second], dim=-1).flatten(-2) if pairs else torch.cat([first, second], dim=-1)
    return torch.cat([y, x[..., rot:]], dim=-1)


def _to_codes(x, cache):
    if cache == 'int8':
        return x.round().clamp(-127, 127).to(torch.int8)
    return x.clamp(-448, 448).to(torch.float8_e4m3fn)


def _append_plain(st, case):
    nh, nkv, page, block, cache = (case[k] for k in ('nh', 'nkv', 'page', 'block', 'cache'))
    turned = _turned(torch.cat([st['q'], st['kn']], dim=1).float(), st)
    live = st['seq'] >= 0
    st['q_out'].copy_(torch.where(live[:, None, None], turned[:, :nh].to(st['q_out'].dtype), st['q_out']))
    row = live.nonzero()[:, 0]
    pos = st['pos'][row].long()
    where = st['table'][st['seq'][row].long(), pos // page].long()
    per = page // block
    at = where * per + pos % page // block                                         # the block of each row
    for name, new in (('k', turned[:, nh:]), ('v', st['vn'].float())):
        pool, scale, new = st[name], st[name + 's'], new[row]
        n = pool.shape[0] * per
        most = torch.zeros((n, nkv), device=DEV).index_reduce_(0, at, new.abs().amax(-1), 'amax')
        touched = torch.zeros(n, dtype=torch.bool, device=DEV).index_fill_(0, at, True)
        begun = torch.zeros(n, dtype=torch.bool, device=DEV).index_fill_(0, at[pos % block == 0], True)
        old = scale.transpose(1, 2).reshape(n, nkv)
        grown = torch.maximum(most / MOST[cache], torch.where(begun[:, None], 0.0, old)).clamp_min(LEAST_SCALE)
        grown = torch.where(touched[:, None], grown, old)
        keep = torch.where(begun[:, None], 1.0, old / grown)
        # what the continued blocks hold, rounded anew
        keep = keep.view(-1, per, nkv).transpose(1, 2)[..., None, None]
        codes = _to_codes((pool.float().unflatten(2, (per, block)) * keep).flatten(2, 3), cache)
        new = _to_codes(new / grown[at][..., None], cache)
        codes = codes.view(torch.uint8)
        codes[where, :, pos % page] = new.view(torch.uint8)
        pool.view(torch.uint8).copy_(codes)
        scale.copy_(grown.view(-1, per, nkv).transpose(1, 2))


def _read_plain(st, case, dtype):
    page, block = case['page'], case['block']
    pos = st['read_pos'].long()
    where = st['table'][st['read_seq'].long(), pos // page].long()
    out = []
    for name in ('k', 'v'):
        x = st[name].view(torch.uint8)[where, :, pos % page].view(st[name].dtype).float()
        out.append((x * st[name + 's'][where, :, pos % page // block][..., None]).to(dtype))
    return out


def _attend_plain(st, case):
    """Every sequence's keys and values gathered to the longest length, scores with a mask, softmax, weighted sum."""
    B, nh, nkv, hd, page, block = (case[k] for k in ('batch', 'nh', 'nkv', 'hd', 'page', 'block'))
    Q, L = st['most_q'], st['most_kv']
    at = torch.arange(L, device=DEV)
    pages = st['table'][:, at // page].clamp_min(0).long()                        # [B, L]
    off = (at % page).expand(B, L)

    def gathered(pool, scale):
        x = pool.view(torch.uint8)[pages, :, off].view(pool.dtype).float()         # [B, L, nkv, hd]
        return x * scale[pages, :, off // block][..., None]
    k = gathered(st['k'], st['ks']).permute(0, 2, 3, 1).contiguous()               # [B, nkv, hd, L]
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
    v = gathered(st['v'], st['vs']).permute(0, 2, 1, 3).contiguous()               # [B, nkv, L, hd]
    o = torch.matmul(e.view(B, nkv, Q * (nh // nkv), L), v).view(B, nkv, Q, nh // nkv, hd) / den.clamp_min(1e-30)
    return o.permute(0, 2, 1, 3, 4).reshape(B, Q, nh, hd)[seq, idx].to(st['q'].dtype)


def _beam_plain(st, case):
    """The 2 K best continuations of each request in order (ties: the lowest beam, then token), and the K best that go on."""
    B, K, V = case['batch'], case['beams'], case['vocab']
    n = 2 * K
    x = st['logits'].float()
    m = x.amax(-1, keepdim=True)
    lse = (x - m).exp().sum(-1, dtype=torch.float64, keepdim=True).log() + m       # (orders of near totals need 64 bits)
    total = ((x - lse) + st['scores'].double().view(B * K, 1)).view(B, K * V)
    return _best_of(total, B, K, V, n, st['eos'])


def _best_of(total, B, K, V, n, eos):
    """The n best of total [B, K V] in 64 bits: (scores, beams, tokens) [B, n] and (scores, rows, tokens) [B, K] of those that do not
    end; -infinity and -1 in places without a continuation."""
    border = total.topk(min(n, K * V), dim=-1).values[:, -1:]
    b, i = ((total >= border) & (total > -torch.inf)).nonzero(as_tuple=True)       # in order of requests, then indexes
    value = total[b, i]
    order = torch.sort(-value, stable=True).indices
    order = order[torch.sort(b[order], stable=True).indices]
    b, i, value = b[order], i[order], value[order]
    starts = torch.searchsorted(b.contiguous(), torch.arange(B, device=total.device))
    rank = torch.arange(len(b), device=total.device) - starts[b]
    b, i, value, rank = (t[rank < n] for t in (b, i, value, rank))

    def placed(width, b, rank, fields):
        out = [torch.full((B, width), -torch.inf, dtype=total.dtype, device=total.device)]
        out += [torch.full((B, width), -1, dtype=torch.int32, device=total.device) for _ in fields[1:]]
        for o, f in zip(out, fields):
            o[b, rank] = f.to(o.dtype)
        return out
    best = placed(n, b, rank, (value, i // V, i % V))
    on = i % V != eos
    count = on.cumsum(0)
    before = torch.cat([count.new_zeros(1), count])[torch.searchsorted(b.contiguous(), torch.arange(B, device=total.device))]
    rank = count - 1 - before[b]
    on &= rank < K
    go = placed(K, b[on], rank[on], (value[on], b[on] * K + i[on] // V, i[on] % V))
    return tuple([best[0].float(), *best[1:], go[0].float(), *go[1:]])


def _held(table, n):
    """How many entries of a table name each of n pages."""
    e = table.reshape(-1).long()
    return torch.zeros(n + 1, dtype=torch.int32, device=DEV).index_add_(0, torch.where(e < 0, n, e), torch.ones_like(e, dtype=torch.int32))[:n]


def _take_pages(st, wanted):
    """Pages for the True places of a mask, the lowest free ones in order; -1 where there are no more."""
    free = (st['holders'] == 0).nonzero()[:, 0]
    rank = wanted.reshape(-1).cumsum(0).view(wanted.shape) - 1
    got = wanted & (rank < free.numel())
    page = torch.where(got, torch.cat([free, free.new_zeros(1)])[rank.clamp(0, free.numel())], -1).int()
    st['missing'] += (wanted & ~got).sum().int()
    st['holders'] += _held(page, st['holders'].numel())
    return page


def _fork_plain(st, case):
    page, table, S = case['page'], st['table'], st['table'].shape[0]
    cols = torch.arange(table.shape[1], device=DEV)
    p = st['parents'].long()
    lens = st['lengths'][p]
    full, rest = lens // page, lens % page
    later = ((p[:, None] == p[None, :]) & torch.ones((S, S), dtype=torch.bool, device=DEV).tril(-1)).any(1)   # not the first child
    new = torch.where((cols < full[:, None]) | ((cols == full[:, None]) & ((rest > 0) & ~later)[:, None]), table[p], -1)
    n = st['holders'].numel()
    st['holders'] += _held(new, n) - _held(table, n)
    dst = _take_pages(st, (rest > 0) & later)
    src = table[p, full.long().clamp_max(table.shape[1] - 1)]
    new = torch.where((cols == full[:, None]) & (dst >= 0)[:, None], dst[:, None], new)
    c = (dst >= 0).nonzero()[:, 0]
    src, dst, rest = src[c].long(), dst[c].long(), rest[c]
    rows = torch.arange(page, device=DEV) < rest[:, None]
    pool = st['pool'].view(torch.uint8) if st['pool'].element_size() == 1 else st['pool']
    pool[:, :, dst] = torch.where(rows[:, None, :, None], pool[:, :, src], pool[:, :, dst])
    if st['scale'] is not None:
        blocks = rows[:, ::case['block']]
        st['scale'][:, :, dst] = torch.where(blocks[:, None], st['scale'][:, :, src], st['scale'][:, :, dst])
    table.copy_(new)
    st['lengths'].copy_(lens)


def _free_plain(st, seqs):
    s = seqs.long()
    st['holders'] -= _held(st['table'][s], st['holders'].numel())
    st['table'][s] = -1
    st['lengths'][s] = 0


def _compact_plain(st):
    used = st['holders'] > 0
    at = torch.arange(used.numel(), device=DEV)
    low = at < used.sum()
    src, dst = (used & ~low).nonzero()[:, 0], (~used & low).nonzero()[:, 0]
    pool = st['pool'].view(torch.uint8) if st['pool'].element_size() == 1 else st['pool']
    pool[:, :, dst] = pool[:, :, src]
    if st['scale'] is not None:
        st['scale'][:, :, dst] = st['scale'][:, :, src]
    to = at.int()
    to[src] = dst.int()
    st['holders'][dst] = st['holders'][src]
    st['holders'][src] = 0
    st['table'].copy_(torch.where(st['table'] >= 0, to[st['table'].clamp_min(0).long()], -1))


def _grow_plain(st, case, counts):
    page = case['page']
    cols = torch.arange(st['table'].shape[1], device=DEV)
    have, want = -(-st['lengths'] // page), -(-(st['lengths'] + counts) // page)
    new = (cols >= have[:, None]) & (cols < want[:, None])
    got = _take_pages(st, new)
    st['table'].copy_(torch.where(new, got, st['table']))
    st['lengths'] += counts


# ------------------------------------------------------------------------------------------------ what a pass needs
def work(case):
    kind = case['kind']
    if kind == 'append':
        counts, starts = _append_lengths(case)
        rows, b, hd = sum(counts), BYTES[case['dtype']], case['hd']
        q, kv = case['nh'] * hd, 2 * case['nkv'] * hd
        blocks = [(a // case['block'], -(-(a + n) // case['block'])) for a, n in zip(starts, counts) if n]
        held = sum(a + n - a // case['block'] * case['block'] for a, n in zip(starts, counts) if n)
        return {'bytes': rows * (2 * q * b + kv * (b + 1)) + held * kv * (1 + min(b, 2)) + 12 * case['rows'] + 8 * held +
                16 * case['nkv'] * sum(e - a for a, e in blocks),
                'flops': 3 * rows * (case['nh'] + case['nkv']) * case['rot'] + 3 * rows * kv + held * kv}
    if kind == 'attend':
        q_lens, kv_lens = _attend_lengths(case)
        whole = case['shared'] // case['page'] * case['page']
        read = case['groups'] * whole + sum(n - whole for n in kv_lens)
        pairs = sum(q * n - q * (q - 1) // 2 for q, n in zip(q_lens, kv_lens))
        return {'bytes': 2 * read * case['nkv'] * (case['hd'] + 4 / case['block']) +
                2 * sum(q_lens) * case['nh'] * case['hd'] * BYTES[case['dtype']],
                'flops': 4 * pairs * case['nh'] * case['hd']}
    if kind == 'beam':
        n = case['batch'] * case['beams']
        return {'bytes': n * case['vocab'] * BYTES[case['dtype']] + n * (4 + 2 * 12 + 12), 'flops': 3 * n * case['vocab']}
    lens, common = _page_lengths(case)
    page, K = case['page'], case['beams']
    scale = 4 / case['block'] if case['cache'] in MOST else 0
    row = 2 * case['layers'] * case['nkv'] * (case['hd'] * BYTES[case['cache']] + scale)
    tables = 8 * len(lens) * K * (-(-max(lens) // page) + 1)
    if kind == 'fork':
        # of the beams drawn towards their request's best, about half continue a beam that another continues too
        return {'bytes': 2 * row * sum(n % page for n in lens) * max(1, K // 2) + tables, 'flops': 0}
    moved = [sum(-(-n // page) for n in lens[i::2]) for i in range(2)]
    return {'bytes': 2 * row * page * min(moved) + tables, 'flops': 0}


# ------------------------------------------------------------------------------------------------ 64-bit results
def exact(case, seed):
    st = prepare(case, seed)
    if case['kind'] == 'append':
        return _append_exact(st, case)
    if case['kind'] == 'attend':
        return _attend_exact(st, case)
    if case['kind'] == 'beam':
        B, K, V = case['batch'], case['beams'], case['vocab']
        total = torch.log_softmax(st['logits'].double(), -1).view(B, K, V) + st['scores'].double()[:, :, None]
        score, go = np.full((B, 2 * K), -np.inf), np.full((B, K), -np.inf)
        for b in range(B):
            flat = total[b].reshape(-1)
            top = flat.topk(min(4 * K, K * V)).values.cpu().numpy()[:2 * K]
            score[b, :len(top)] = top
            flat[st['eos']::V] = -torch.inf
            best = flat.topk(min(K, K * V)).values.cpu().numpy()
            # (of the 2 K best: as many go on as do not end)
            best = best[best >= top[-1]] if np.isfinite(top[-1]) else best
            go[b, :len(best)] = best
        return (torch.from_numpy(score), None, None, torch.from_numpy(go), None, None)
    return _pages_exact(st, case)


def _append_exact(st, case):
    nh, page, block, rot = (case[k] for k in ('nh', 'page', 'block', 'rot'))
    j = np.arange(rot // 2)
    turn = torch.from_numpy(np.exp(1j * st['pos'].cpu().numpy()[:, None].astype(np.float64) * np.exp(-np.log(THETA) * 2 * j / rot)))
    x = torch.cat([st['q'], st['kn']], 1).double().cpu()
    one, two = (slice(0, rot, 2), slice(1, rot, 2)) if case['pairs'] else (slice(0, rot // 2), slice(rot // 2, rot))
    z = torch.complex(x[..., one], x[..., two]) * turn[:, None]
    x[..., one], x[..., two] = z.real, z.imag
    seq, pos, table = st['seq'].tolist(), st['pos'].tolist(), st['table'].tolist()
    q = st['q_out'].double().cpu()
    groups = {}
    for r, (s, p) in enumerate(zip(seq, pos)):
        if s >= 0:
            q[r] = x[r, :nh]
            groups.setdefault((table[s][p // page], p % page // block), []).append(r)
    out = {'q': q}
    for name, new in (('k', x[:, nh:].numpy()), ('v', st['vn'].double().cpu().numpy())):
        codes, scale = st[name].cpu().float().double().numpy(), st[name + 's'].double().cpu().numpy()
        for (e, b), rows in groups.items():
            begun = any(pos[r] % block == 0 for r in rows)
            old = np.zeros_like(scale[e, :, b]) if begun else scale[e, :, b]
            grown = np.maximum(np.maximum(np.abs(new[rows]).max((0, 2)) / MOST[case['cache']], old), LEAST_SCALE)
            part = slice(b * block, (b + 1) * block)
            if not begun:
                codes[e, :, part] = _rounded(codes[e, :, part] * (old / grown)[:, None, None], case['cache'])
            for r in rows:
                codes[e, :, pos[r] % page] = _rounded(new[r] / grown[:, None], case['cache'])
            scale[e, :, b] = grown
        held = [(table[s][p // page], p % page) for s, p in zip(st['read_seq'].tolist(), st['read_pos'].tolist())]
        out[name] = torch.from_numpy(np.stack([codes[e, :, i] * scale[e, :, i // block, None] for e, i in held])
                                     if held else np.zeros((0, *codes.shape[1::2])))
        out[name + 's'] = torch.from_numpy(scale)
    return out


def _rounded(x, cache):
    """The nearest code, ties to even: a whole number up to 127, or 3 fraction bits with exponents from -6, up to 448."""
    if cache == 'int8':
        return np.clip(np.rint(x), -127, 127)
    x = np.clip(x, -448, 448)
    step = np.exp2(np.floor(np.log2(np.maximum(np.abs(x), 2.0 ** -6))) - 3)
    return np.rint(x / step) * step


def _attend_exact(st, case):
    nh, nkv, hd, page = case['nh'], case['nkv'], case['hd'], case['page']
    out, r0 = torch.zeros((sum(st['q_lens']), nh, hd), dtype=torch.float64, device=DEV), 0
    for s, (nq, n) in enumerate(zip(st['q_lens'], st['kv_lens'])):
        pages = st['table'][s, :-(-n // page)].long()
        rows = []
        for pool, scale in ((st['k'], st['ks']), (st['v'], st['vs'])):
            x = pool.view(torch.uint8)[pages].view(pool.dtype).double()
            x *= scale[pages].double().repeat_interleave(case['block'], -1)[..., None]
            rows.append(x.permute(1, 0, 2, 3).reshape(nkv, -1, hd)[:, :n])
        hidden = torch.arange(n, device=DEV)[None, :] > torch.arange(n - nq, n, device=DEV)[:, None]
        for h in range(nh):
            kv = h // (nh // nkv)
            w = st['q'][r0:r0 + nq, h].double() @ rows[0][kv].T.contiguous() / hd ** 0.5
            w = torch.softmax(w.masked_fill(hidden, -torch.inf), dim=-1)
            out[r0:r0 + nq, h] = w @ rows[1][kv].contiguous()
        r0 += nq
    return out


def _pages_exact(st, case):
    """The tables as lists, page by page."""
    page, pool, scale = case['page'], st['pool'], st['scale']
    pool = pool.view(torch.uint8) if pool.element_size() == 1 else pool
    table, lens = [[e for e in row if e >= 0] for row in st['table'].tolist()], st['lengths'].tolist()
    holders, width = st['holders'].tolist(), st['table'].shape[1]

    def lowest():
        e = holders.index(0)
        holders[e] = 1
        return e

    def copy(src, dst, rows):
        if src:
            src, dst = torch.tensor(src, device=DEV), torch.tensor(dst, device=DEV)
            for i in range(rows[0] if len(set(rows)) == 1 else page):
                some = torch.tensor([r > i for r in rows], device=DEV)
                pool[:, :, dst[some], :, i] = pool[:, :, src[some], :, i]
                if scale is not None and i % case['block'] == 0:
                    scale[:, :, dst[some], :, i // case['block']] = scale[:, :, src[some], :, i // case['block']]
    if case['kind'] == 'fork':
        parents, seen, new, copies = st['parents'].tolist(), set(), [], []
        for p in parents:
            rest = lens[p] % page
            new.append(list(table[p]) if p not in seen or not rest else table[p][:-1] + [None])
            seen.add(p)
        for row in table:
            for e in row:
                holders[e] -= 1
        for row in new:
            for e in row:
                if e is not None:
                    holders[e] += 1
        for s, row in enumerate(new):
            if row and row[-1] is None:
                row[-1] = lowest()
                copies.append((table[parents[s]][-1], row[-1], lens[parents[s]] % page))
        copy(*([c[i] for c in copies] for i in range(3)))
        table, lens = new, [lens[p] for p in parents]
    else:
        for s in st['ends'][0].tolist():
            for e in table[s]:
                holders[e] -= 1
            table[s], lens[s] = [], 0
        used = [e for e, h in enumerate(holders) if h]
        high = [e for e in used if e >= len(used)]
        low = [e for e, h in enumerate(holders) if not h][:len(high)]
        copy(high, low, [page] * len(high))
        to = dict(zip(high, low))
        table = [[to.get(e, e) for e in row] for row in table]
        for e, f in to.items():
            holders[f], holders[e] = holders[e], 0
        for s, n in enumerate(st['begins'][0].tolist()):
            table[s] += [lowest() for _ in range(-(-(lens[s] + n) // page) - len(table[s]))]
            lens[s] += n
    out = {'table': _int([row + [-1] * (width - len(row)) for row in table]), 'lengths': _int(lens), 'holders': _int(holders),
           'missing': None, 'pool': st['pool'], 'scale': scale}
    return {k: None if v is None else v if v.dtype in (torch.int32, torch.int8) else v.double() for k, v in out.items()}
