"""Attention between the MoE blocks, as cases that can be timed: the norms of queries and
keys with the position rotation, the append of keys and values to a paged cache, and the
attention of new tokens over that cache.

With `own` false, `run` computes each operator in elementary torch operations in 32 bits
(angles in 64), over sequences padded to the longest; with `own` true it makes the calls a
program makes.  `exact` restates the operators in 64 bits, sequence by sequence.
"""
import math
import random

import torch

own = False

DTYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16}
EPS = 1e-6

# (query heads, key-value heads, head size, rotated channels): heads of 256 of which a quarter is
# rotated, as the hidden-2048 model's projections of 4096 have them; grouped heads of 128;
# one key-value head; a head for each query head; an odd group.
HEADS = [(16, 2, 256, 64), (32, 8, 128, 128), (8, 1, 256, 64), (16, 16, 64, 64), (12, 4, 128, 64),
         (20, 4, 64, 32)]


def _heads(i):
    hq, hk, d, r = HEADS[i]
    return dict(hq=hq, hk=hk, d=d, rot=r)


def _attend(name, spread, sequences, new, context, page, heads, dtype='bf16', gate=True, pad=0):
    return dict(name=name, kind='attention', sequences=sequences, new_min=new[0], new_max=new[1],
                context_min=context[0], context_max=context[1], page=page, dtype=dtype,
                spread=spread, gate=gate, pad=pad, **_heads(heads))


def listed():
    return [
        # one decode step's queries and keys: latency alone
        dict(name='norm_1', kind='norm', tokens=1, start=9000, dtype='bf16', **_heads(0)),
        # a short prompt of a model with fully rotated heads of 128, fp16
        dict(name='norm_333_fp16', kind='norm', tokens=333, start=0, dtype='fp16', **_heads(1)),
        # a prefill chunk far into a long prompt
        dict(name='norm_4096', kind='norm', tokens=4096, start=200000, dtype='bf16', **_heads(0)),
        # a decode step of 64 users: one token each to its own page
        dict(name='append_64', kind='append', sequences=64, new_min=1, new_max=1, context_min=100,
             context_max=1000, page=64, dtype='bf16', spread=1, **_heads(0)),
        # chunks of several prompts at once, small pages that the chunks do not fill, fp16
        dict(name='append_mixed_fp16', kind='append', sequences=9, new_min=30, new_max=900,
             context_min=0, context_max=500, page=16, dtype='fp16', spread=2, **_heads(1)),
        # one user's decode step at a short context: the smallest attention call
        _attend('decode_1', 3, 1, (1, 1), (999, 999), 64, 0),
        # one user's decode step at the end of a very long context
        _attend('decode_long', 4, 1, (1, 1), (262143, 262143), 64, 0),
        # a decode step of 64 users whose contexts differ by a factor of 32, one padded row
        _attend('decode_64', 5, 64, (1, 1), (400, 13000), 64, 0, pad=1),
        # the first chunk of a prompt: the causal triangle
        _attend('chunk_first', 6, 1, (2048, 2048), (0, 0), 64, 0),
        # a later chunk of a long prompt: the largest product
        _attend('chunk_late', 7, 1, (2048, 2048), (8192, 8192), 64, 0),
        # prompts and single tokens in one call, small pages, fp16, heads of 128
        _attend('mixed_fp16', 8, 12, (1, 700), (0, 3000), 16, 1, 'fp16', gate=False, pad=5),
        # several short drafts verified against their contexts, a head for each query head
        _attend('verify_24', 9, 24, (2, 9), (300, 5000), 32, 3, gate=False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5))))))


def _range(name, rng, lo, hi):
    lo, hi = sorted((_log_int(rng, lo, hi), _log_int(rng, lo, hi)))
    return {name + '_min': lo, name + '_max': hi}


def draw(rng):
    kind = rng.choice(['norm', 'append', 'attention', 'attention', 'attention'])
    case = dict(kind=kind, dtype=rng.choice(['bf16', 'bf16', 'fp16']),
                **_heads(rng.randrange(len(HEADS))))
    if kind == 'norm':
        return dict(case, tokens=_log_int(rng, 1, 4096),
                    start=rng.choice([0, _log_int(rng, 1, 250000)]))
    case.update(page=rng.choice([16, 32, 64, 128]), spread=rng.randrange(1 << 20))
    if kind == 'append':
        sequences = _log_int(rng, 1, 64)
        return dict(case, sequences=sequences, **_range('new', rng, 1, 4096 // sequences),
                    **_range('context', rng, 1, 1000))
    case.update(gate=rng.random() < 0.5, pad=rng.choice([0, 0, 3]))
    form = rng.choice(['decode', 'chunk', 'few'])
    if form == 'decode':
        sequences = _log_int(rng, 1, 64)
        return dict(case, sequences=sequences, new_min=1, new_max=1,
                    **_range('context', rng, 1, min(100000, 400000 // sequences)))
    if form == 'few':
        sequences = _log_int(rng, 1, 24)
        return dict(case, sequences=sequences, **_range('new', rng, 1, 24),
                    **_range('context', rng, 1, 5000))
    sequences = rng.choice([1, 1, 2, 5])
    return dict(case, sequences=sequences, **_range('new', rng, 25, 2048 // sequences),
                **_range('context', rng, 1, 8192 // sequences))


# ------------------------------------------------------------------ inputs
def _lengths(case):
    """(new tokens, context after them) of each sequence, by the case alone."""
    rng = random.Random(case['spread'])

    def pick(name):
        lo, hi = case[name + '_min'], case[name + '_max']
        return lo if lo == hi else max(lo, min(hi, round(math.exp(
            rng.uniform(math.log(max(lo, 1)), math.log(hi))))))

    out = []
    for _ in range(case['sequences']):
        new = pick('new')
        out.append((new, pick('context') + new))
    return out


def _tokens(case):
    if case['kind'] == 'norm':
        return case['tokens']
    return sum(n for n, _ in _lengths(case)) + case.get('pad', 0)


def _inputs(case, seed):
    g = torch.Generator(device='cuda')
    g.manual_seed((seed * 1_000_003 + sum(map(ord, case['kind'])) * 7919) % (2 ** 62))
    dt, t = DTYPES[case['dtype']], _tokens(case)
    hq, hk, d, rot = case['hq'], case['hk'], case['d'], case['rot']

    def rows(heads, scale=1.0):
        return (torch.randn(t, heads, d, generator=g, device='cuda') * scale).to(dt)

    st = dict(kind=case['kind'], eps=EPS)
    if case['kind'] in ('norm', 'append'):
        # projections before their norm: rows of different magnitudes; the query projection of a
        # model with gated attention holds a query and a gate of each head side by side
        st['q'] = torch.cat([rows(hq, 3.0), rows(hq)], -1)[..., :d]
        st['k'], st['v'] = rows(hk, 3.0), rows(hk)
        st['q_weight'] = torch.randn(d, generator=g, device='cuda') * 0.1
        st['k_weight'] = torch.randn(d, generator=g, device='cuda') * 0.1
        j = torch.arange(rot // 2, device='cuda', dtype=torch.float64)
        st['inv_freq'] = (1e7 ** (-2.0 * j / rot)).to(torch.float32)
    if case['kind'] == 'norm':
        st['positions'] = torch.arange(t, device='cuda') + case['start']
        return st
    new, length = zip(*_lengths(case))
    page, s = case['page'], len(new)
    need = [-(-n // page) for n in length]
    pages = sum(need) + 2
    order = torch.randperm(pages, generator=g, device='cuda').to(torch.int32)
    table = torch.zeros(s, max(need), dtype=torch.int32)
    place = torch.arange(max(need))
    first = torch.tensor([0] + need).cumsum(0)[:s]
    index = torch.where(place < torch.tensor(need)[:, None], first[:, None] + place, 0)
    st['table'] = order[index.to('cuda')].contiguous()
    st['starts'] = torch.tensor([0] + list(new)).cumsum(0).to('cuda', torch.int32)
    st['lengths'] = torch.tensor(length).to('cuda', torch.int32)
    st['max_new'] = max(new)
    # keys as they are after their norm and rotation; values as projected
    st['k_pages'] = torch.randn(pages, hk, page, d, generator=g, device='cuda', dtype=dt)
    st['v_pages'] = torch.randn(pages, hk, page, d, generator=g, device='cuda', dtype=dt)
    if case['kind'] == 'attention':
        st['q'] = rows(hq, 1.5)
        st['gate'] = torch.cat([rows(hq), rows(hq, 2.0)], -1)[..., d:] if case['gate'] else None
        st['out'] = torch.zeros(t, hq, d, device='cuda', dtype=dt)
    return st


def prepare(case, seed):
    return _inputs(case, seed)


# ------------------------------------------------------------------ one pass
def _norm_rope(x, weight, positions, inv_freq, eps):
    v = x.float()
    v = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + eps) * (1.0 + weight)
    angle = positions.double()[:, None] * inv_freq.double()
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    half = inv_freq.shape[0]
    a, b, rest = v[..., :half], v[..., half:2 * half], v[..., 2 * half:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1).to(x.dtype)


def _places(st):
    """(sequence, place among its new tokens, position in its context) of every row of q."""
    starts, rows = st['starts'].long(), torch.arange(st['q'].shape[0], device='cuda')
    seq = (torch.searchsorted(starts, rows, right=True) - 1).clamp(max=starts.shape[0] - 2)
    place = rows - starts[seq]
    return seq, place, st['lengths'].long()[seq] - (starts[seq + 1] - starts[seq]) + place


def _attention(st):
    q, k_pages, v_pages, table = st['q'], st['k_pages'], st['v_pages'], st['table'].long()
    t, hq, d = q.shape
    s, hk, n = table.shape[0], k_pages.shape[1], st['max_new']
    g, keys = hq // hk, table.shape[1] * k_pages.shape[2]
    starts, lengths = st['starts'].long(), st['lengths'].long()
    new = starts[1:] - starts[:-1]
    step = torch.arange(n, device='cuda')
    rows = (starts[:-1, None] + step).clamp(max=t - 1)
    queries = q[rows].float().view(s, n, hk, g, d).transpose(1, 2).reshape(s * hk, n * g, d)
    key = torch.arange(keys, device='cuda')
    k = k_pages[table].transpose(1, 2).reshape(s * hk, keys, d).float()
    scores = torch.bmm(queries, k.transpose(1, 2)).mul_(d ** -0.5).view(s, hk, n, g, keys)
    seen = key <= (lengths - new)[:, None, None] + step[:, None]  # [s, n, keys]
    scores.masked_fill_(~(seen & (key < lengths[:, None, None]))[:, None, :, None], float('-inf'))
    p = torch.exp(scores - scores.amax(-1, keepdim=True).clamp_min(-1e30))
    total = p.sum(-1, keepdim=True)
    v = torch.where((key < lengths[:, None])[:, None, :, None],
                    v_pages[table].transpose(1, 2).reshape(s, hk, keys, d).float(), 0.0)
    o = torch.bmm(p.view(s * hk, n * g, keys), v.view(s * hk, keys, d)).view(s, hk, n, g, d)
    o = torch.where(total > 0, o / total, 0.0).transpose(1, 2).reshape(s, n, hq, d)
    seq, place, _ = _places(st)
    o = o[seq, place.clamp(max=n - 1)]
    if st['gate'] is not None:
        o = o / (1.0 + torch.exp(-st['gate'].float()))
    live = torch.arange(t, device='cuda') < starts[-1]
    return torch.where(live[:, None, None], o.to(q.dtype), st['out'])


def run(state):
    st = state
    if own:
        from localmoe35ba3b_amd.operators import attention
        if st['kind'] == 'norm':
            return attention.qk_norm_rope(st['q'], st['k'], st['q_weight'], st['k_weight'],
                                          st['positions'], st['inv_freq'], st['eps'])
        if st['kind'] == 'append':
            q = attention.append(st['k_pages'], st['v_pages'], st['k'], st['v'], st['starts'],
                                 st['lengths'], st['table'], inv_freq=st['inv_freq'],
                                 k_weight=st['k_weight'], q=st['q'], q_weight=st['q_weight'],
                                 eps=st['eps'])
            return q, st['k_pages'], st['v_pages']
        return attention.paged_attention(st['q'], st['k_pages'], st['v_pages'], st['starts'],
                                         st['lengths'], st['table'], gate=st['gate'],
                                         max_new=st['max_new'], out=st['out'])
    if st['kind'] == 'norm':
        args = st['positions'], st['inv_freq'], st['eps']
        return tuple(_norm_rope(st[n], st[n + '_weight'], *args) for n in ('q', 'k'))
    if st['kind'] == 'append':
        seq, _, position = _places(st)
        page = st['k_pages'].shape[2]
        at = (st['table'].long()[seq, position // page][:, None],
              torch.arange(st['k'].shape[1], device='cuda'), (position % page)[:, None])
        args = position, st['inv_freq'], st['eps']
        st['k_pages'][at] = _norm_rope(st['k'], st['k_weight'], *args)
        st['v_pages'][at] = st['v']
        return _norm_rope(st['q'], st['q_weight'], *args), st['k_pages'], st['v_pages']
    return _attention(st)


# ------------------------------------------------------------------ work
def work(case):
    hq, hk, d = case['hq'], case['hk'], case['d']
    if case['kind'] == 'norm':
        elements = _tokens(case) * (hq + hk) * d
        return dict(bytes=4 * elements + 8 * _tokens(case) + 8 * d, flops=8 * elements)
    if case['kind'] == 'append':
        t = _tokens(case)
        return dict(bytes=4 * t * (hq + 2 * hk) * d + 8 * d, flops=8 * t * (hq + hk) * d)
    lengths = _lengths(case)
    rows = sum(n for n, _ in lengths)
    pairs = sum(n * (l - n) + n * (n + 1) // 2 for n, l in lengths)
    return dict(bytes=2 * d * ((3 if case['gate'] else 2) * rows * hq
                               + 2 * hk * sum(l for _, l in lengths)),
                flops=4 * hq * d * pairs)


# ------------------------------------------------------------------ 64-bit results
def _exact_rows(x, weight, positions, inv_freq):
    """Pairs (i, i + half) of the normalized row as complex numbers, turned by the angle."""
    z = x.double()
    z = z / (z.square().sum(-1, keepdim=True) / z.shape[-1] + EPS).sqrt()
    z = z + z * weight.double()
    half = inv_freq.shape[0]
    turn = torch.polar(torch.ones((), dtype=torch.float64, device='cuda'),
                       torch.outer(positions.double(), inv_freq.double()))
    pair = torch.complex(z[..., :half].contiguous(),
                         z[..., half:2 * half].contiguous()) * turn[:, None]
    z[..., :half], z[..., half:2 * half] = pair.real, pair.imag
    return z


def exact(case, seed):
    st = _inputs(case, seed)
    if case['kind'] == 'norm':
        return tuple(_exact_rows(st[n], st[n + '_weight'], st['positions'], st['inv_freq'])
                     for n in ('q', 'k'))
    page, table, row = case['page'], st['table'].tolist(), 0
    if case['kind'] == 'append':
        position = torch.cat([torch.arange(l - n, l) for n, l in _lengths(case)]).to('cuda')
        q, k = (_exact_rows(st[n], st[n + '_weight'], position, st['inv_freq'])
                for n in ('q', 'k'))
        k_pages, v_pages = st['k_pages'].double(), st['v_pages'].double()
        for s, (n, l) in enumerate(_lengths(case)):
            p = l - n
            while p < l:  # the part of one page
                m = min(page - p % page, l - p)
                to = (table[s][p // page], slice(None), slice(p % page, p % page + m))
                k_pages[to] = k[row:row + m].transpose(0, 1)
                v_pages[to] = st['v'][row:row + m].transpose(0, 1).double()
                p, row = p + m, row + m
        return q, k_pages, v_pages
    out, g = st['out'].double(), case['hq'] // case['hk']
    for s, (n, l) in enumerate(_lengths(case)):
        used = table[s][:-(-l // page)]
        for h in range(case['hk']):
            k = st['k_pages'][used, h].reshape(-1, case['d'])[:l].double()
            v = st['v_pages'][used, h].reshape(-1, case['d'])[:l].double()
            for a in range(0, n, 256):
                b = min(n, a + 256)
                q = st['q'][row + a:row + b, h * g:(h + 1) * g].double()
                w = (q.reshape(-1, case['d']) @ k.t()).view(b - a, g, l) / math.sqrt(case['d'])
                last = torch.arange(l - n + a, l - n + b, device='cuda')[:, None, None]
                w = w.masked_fill(torch.arange(l, device='cuda') > last, float('-inf'))
                w = torch.softmax(w, -1).view(-1, l)
                out[row + a:row + b, h * g:(h + 1) * g] = (w @ v).view(b - a, g, -1)
        row += n
    if case['gate']:
        out[:row] *= torch.sigmoid(st['gate'][:row].double())
    return out
