"""Attention over a cache held in 8 bits and what feeds it, as cases that can be timed: the norms of
queries and keys with a rotation by positions of several axes, the append to an e4m3 cache with a
scale for each 16 positions of a head, attention over that cache, and the norm of rows after the
residual's addition that leaves them in 8 bits for a W8A8 product.

With `own` false, `run` computes each operator in elementary torch operations in 32 bits (angles in
64), over sequences padded to the longest; with `own` true it makes the calls a program makes.
`exact` restates the operators in 64 bits, sequence by sequence.  What is held in 8 bits is returned
as the values it stands for, in the type of the rows (exact for the cache: e4m3 times a power of two).
"""
import math
import random

import torch

own = False

DTYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16}
E4M3 = torch.float8_e4m3fn
EPS = 1e-6
BLOCK = 16  # positions of a head that share a scale
LEAST = {torch.bfloat16: -117, torch.float16: -15}  # exponent of the smallest scale
MOST = {torch.bfloat16: 1.875 * 2.0 ** 127, torch.float16: 61440.0}  # largest value held

# (query heads, key-value heads, head size, rotated channels): heads of 256 of which a quarter is
# rotated, as the hidden-2048 model's projections of 4096 have them; grouped heads of 128;
# one key-value head; a head for each query head; an odd group.
HEADS = [(16, 2, 256, 64), (32, 8, 128, 128), (8, 1, 256, 64), (16, 16, 64, 64), (12, 4, 128, 64),
         (20, 4, 64, 32)]


def _heads(i):
    hq, hk, d, r = HEADS[i]
    return dict(hq=hq, hk=hk, d=d, rot=r)


def _append(name, spread, sequences, new, context, prefix, page, heads, dtype='bf16', axes=1):
    return dict(name=name, kind='append', sequences=sequences, new_min=new[0], new_max=new[1],
                context_min=context[0], context_max=context[1], prefix=prefix, page=page,
                spread=spread, axes=axes, dtype=dtype, **_heads(heads))


def _attend(name, spread, sequences, new, context, page, heads, dtype='bf16', gate=True, pad=0):
    return dict(name=name, kind='attention', sequences=sequences, new_min=new[0], new_max=new[1],
                context_min=context[0], context_max=context[1], page=page, dtype=dtype,
                spread=spread, gate=gate, pad=pad, **_heads(heads))


def listed():
    return [
        # one decode step of a prompt with images: latency alone
        dict(name='rotate_1', kind='rotate', tokens=1, start=9000, axes=3, dtype='bf16',
             **_heads(0)),
        # text and images of a long prompt's chunk, every channel rotated, fp16
        dict(name='rotate_2999_fp16', kind='rotate', tokens=2999, start=5000, axes=3,
             dtype='fp16', **_heads(1)),
        # a decode step of 64 users behind a prompt that they share, each with pages of its own
        _append('append_64', 1, 64, (1, 1), (1, 60), 512, 64, 0),
        # chunks of several prompts that end inside blocks and small pages, fp16
        _append('append_mixed_fp16', 2, 9, (30, 900), (1, 100), 0, 16, 1, 'fp16'),
        # a prefill chunk with images
        _append('append_4096', 3, 1, (4096, 4096), (1000, 1000), 992, 64, 0, axes=3),
        # one user's decode step at a short context: the smallest attention call
        _attend('decode_1', 4, 1, (1, 1), (999, 999), 64, 0),
        # one user's decode step at the end of a very long context
        _attend('decode_long', 5, 1, (1, 1), (262143, 262143), 64, 0),
        # a decode step of 64 users whose contexts differ by a factor of 32, one padded row
        _attend('decode_64', 6, 64, (1, 1), (400, 13000), 64, 0, pad=1),
        # a later chunk of a long prompt: the largest product
        _attend('chunk_late', 7, 1, (2048, 2048), (8192, 8192), 64, 0),
        # prompts and single tokens in one call, small pages, fp16, heads of 128
        _attend('mixed_fp16', 8, 12, (1, 700), (1, 3000), 16, 1, 'fp16', gate=False, pad=5),
        # the row of a decode step on its way into a W8A8 projection
        dict(name='norm_1', kind='norm', tokens=1, hidden=2048, dtype='bf16'),
        # the same of a prefill chunk
        dict(name='norm_2048', kind='norm', tokens=2048, hidden=2048, dtype='bf16'),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5))))))


def _range(name, rng, lo, hi):
    lo, hi = sorted((_log_int(rng, lo, hi), _log_int(rng, lo, hi)))
    return {name + '_min': lo, name + '_max': hi}


def draw(rng):
    kind = rng.choice(['rotate', 'append', 'attention', 'attention', 'attention', 'norm'])
    case = dict(kind=kind, dtype=rng.choice(['bf16', 'bf16', 'fp16']))
    if kind == 'norm':
        return dict(case, tokens=_log_int(rng, 1, 4096), hidden=128 * _log_int(rng, 4, 64))
    case.update(_heads(rng.randrange(len(HEADS))))
    if kind == 'rotate':
        return dict(case, tokens=_log_int(rng, 1, 4096), axes=rng.choice([2, 3, 3]),
                    start=rng.choice([0, _log_int(rng, 1, 250000)]))
    case.update(page=rng.choice([16, 32, 64, 128]), spread=rng.randrange(1 << 20))
    if kind == 'append':
        sequences = _log_int(rng, 1, 64)
        return dict(case, sequences=sequences, prefix=rng.choice([0, 0, 256]),
                    axes=rng.choice([1, 1, 3]), **_range('new', rng, 1, 4096 // sequences),
                    **_range('context', rng, 1, 200))
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
            rng.uniform(math.log(lo), math.log(hi))))))

    out = []
    for _ in range(case['sequences']):
        new = pick('new')
        out.append((new, case.get('prefix', 0) + pick('context') + new))
    return out


def _tokens(case):
    if 'tokens' in case:
        return case['tokens']
    return sum(n for n, _ in _lengths(case)) + case.get('pad', 0)


def _grid(at, axes):
    """Positions on `axes` axes of the tokens at places `at` of a prompt in which 100 of 884 tokens
    are text and the others an image, 28 patches a row."""
    inside = at % 884 - 100
    first = at - inside.clamp(min=0)
    row = torch.where(inside < 0, first, first + inside // 28)
    column = torch.where(inside < 0, first, first + inside % 28)
    return torch.stack([first, row, column][:axes] if axes > 1 else [at])


def _blocks(scales):
    """Scales [pages, heads, 2, blocks] as they multiply keys and values [2, pages, heads, blocks,
    BLOCK, dim]."""
    return scales.permute(2, 0, 1, 3)[..., None, None]


def _held(st):
    """Keys and values that the cache holds, [2, pages, heads, page, dim] in the rows' type."""
    kv = st['kv']
    two, pages, heads, page, dim = kv.shape
    values = kv.view(two, pages, heads, page // BLOCK, BLOCK, dim).to(st['dtype'])
    return values.mul_(_blocks(st['scales'])).view(kv.shape)


def _inputs(case, seed):
    g = torch.Generator(device='cuda')
    g.manual_seed((seed * 1_000_003 + sum(map(ord, case['kind'])) * 7919) % (2 ** 62))
    dt, t = DTYPES[case['dtype']], _tokens(case)

    def rows(*shape, scale=1.0):
        return (torch.randn(t, *shape, generator=g, device='cuda') * scale).to(dt)

    st = dict(kind=case['kind'], eps=EPS, dtype=dt)
    if case['kind'] == 'norm':
        # a residual stream larger than what a block adds, with a few strong channels
        hidden = case['hidden']
        st['h'], st['x'] = rows(hidden, scale=4.0), rows(hidden)
        st['h'][:, torch.randint(hidden, (4,), generator=g, device='cuda')] *= 20.0
        st['weight'] = torch.randn(hidden, generator=g, device='cuda') * 0.1
        return st
    hq, hk, d, rot = case['hq'], case['hk'], case['d'], case['rot']
    if case['kind'] != 'attention':
        # projections before their norm: rows of different magnitudes; the query projection of a
        # model with gated attention holds a query and a gate of each head side by side
        st['q'] = torch.cat([rows(hq, d, scale=3.0), rows(hq, d)], -1)[..., :d]
        st['k'], st['v'] = rows(hk, d, scale=3.0), rows(hk, d)
        st['q_weight'] = torch.randn(d, generator=g, device='cuda') * 0.1
        st['k_weight'] = torch.randn(d, generator=g, device='cuda') * 0.1
        j = torch.arange(rot // 2, device='cuda')
        st['inv_freq'] = (1e7 ** (-2.0 * j.double() / rot)).to(torch.float32)
        # pairs take the axes in turn, as far as the others reach
        st['axes'] = torch.where(j < rot // 2 - 2, j % case['axes'], 0).to(torch.int32)
        if case['kind'] == 'rotate':
            st['positions'] = _grid(torch.arange(t, device='cuda') + case['start'], case['axes'])
            return st
    new, length = zip(*_lengths(case))
    page, s = case['page'], len(new)
    shared = case.get('prefix', 0) // page  # whole pages that all sequences read
    need = [-(-n // page) for n in length]
    pages = sum(need) - shared * (s - 1) + 2
    order = torch.randperm(pages, generator=g, device='cuda').to(torch.int32)
    place = torch.arange(max(need))
    first = torch.tensor([0] + [n - shared for n in need]).cumsum(0)[:s]
    index = torch.where(place < shared, place, first[:, None] + place)
    index = torch.where(place < torch.tensor(need)[:, None], index, 0)
    st['table'] = order[index.to('cuda')].contiguous()
    st['starts'] = torch.tensor([0] + list(new)).cumsum(0).to('cuda', torch.int32)
    st['lengths'] = torch.tensor(length).to('cuda', torch.int32)
    st['max_new'] = max(new)
    # keys as they are after their norm and rotation, values as projected, in 8 bits; blocks of
    # different magnitudes
    nb = page // BLOCK
    kv = torch.empty(2, pages, hk, page, d, device='cuda', dtype=E4M3)
    st['scales'] = torch.empty(pages, hk, 2, nb, device='cuda')
    for side in range(2):
        x = torch.randn(pages, hk, nb, BLOCK, d, generator=g, device='cuda', dtype=dt).float()
        x *= torch.rand(pages, hk, nb, 1, 1, generator=g, device='cuda') + 0.5
        scale = _scale(x.abs().amax((-1, -2)), dt)
        kv[side] = (x / scale[..., None, None]).to(E4M3).view(pages, hk, page, d)
        st['scales'][:, :, side] = scale
    st['kv'] = kv
    if case['kind'] == 'append':
        st['positions'] = None
        if case['axes'] > 1:
            at = torch.cat([torch.arange(n - m, n) for m, n in zip(new, length)]).to('cuda')
            st['positions'] = _grid(at, case['axes'])
        return st
    st['q'] = rows(hq, d, scale=1.5)
    st['gate'] = (torch.cat([rows(hq, d), rows(hq, d, scale=2.0)], -1)[..., d:] if case['gate']
                  else None)
    st['out'] = torch.zeros(t, hq, d, device='cuda', dtype=dt)
    return st


def prepare(case, seed):
    return _inputs(case, seed)


# ------------------------------------------------------------------ one pass
def _scale(amax, dt):
    """The smallest power of two that brings amax to at most 448."""
    m, e = torch.frexp(amax.clamp(max=MOST[dt]))
    e = torch.where(m > 0.875, e - 8, e - 9)
    return torch.ldexp(torch.ones_like(amax), e.clamp(min=LEAST[dt]))


def _norm_rope(x, weight, positions, axes, inv_freq, eps):
    v = x.float()
    v = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + eps) * (1.0 + weight)
    angle = positions.t().double()[:, axes.long()] * inv_freq.double()
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    half = inv_freq.shape[0]
    a, b, rest = v[..., :half], v[..., half:2 * half], v[..., 2 * half:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)


def _places(st):
    """(sequence, place among its new tokens, position in its context) of every row of q."""
    starts, rows = st['starts'].long(), torch.arange(st['q'].shape[0], device='cuda')
    seq = (torch.searchsorted(starts, rows, right=True) - 1).clamp(max=starts.shape[0] - 2)
    place = rows - starts[seq]
    return seq, place, st['lengths'].long()[seq] - (starts[seq + 1] - starts[seq]) + place


def _append_plain(st):
    kv, scales, dt = st['kv'], st['scales'], st['dtype']
    _, pages, heads, page, dim = kv.shape
    nb = page // BLOCK
    seq, _, at = _places(st)
    positions = at[None] if st['positions'] is None else st['positions']
    args = positions, st['axes'], st['inv_freq'], st['eps']
    rows = torch.stack([_norm_rope(st['k'], st['k_weight'], *args), st['v'].float()], 2)
    rows = rows.clamp(-MOST[dt], MOST[dt])  # [tokens, heads, 2, dim]
    number = st['table'].long()[seq, at // page]
    block = number * nb + at % page // BLOCK  # of the whole cache
    amax = torch.zeros(pages * nb, heads, 2, device='cuda')
    amax.index_reduce_(0, block, rows.abs().amax(-1), 'amax')
    # the first new row of every block, BLOCK of one without any: rows before it are held already,
    # rows behind the last keep their bytes
    first = torch.full((pages * nb,), float(BLOCK), device='cuda').index_reduce_(
        0, block, (at % BLOCK).float(), 'amin')[:, None, None]
    old = scales.permute(0, 3, 1, 2).reshape(pages * nb, heads, 2)
    scale = torch.maximum(torch.where(first > 0, old, 0.0), _scale(amax, dt))
    scale = torch.where(first < BLOCK, scale, old)
    ratio = torch.where(torch.arange(BLOCK, device='cuda') < first[..., None],
                        (old / scale)[..., None], 1.0)  # [blocks, heads, 2, BLOCK]
    ratio = ratio.view(pages, nb, heads, 2, BLOCK).permute(3, 0, 2, 1, 4)[..., None]
    values = kv.view(2, pages, heads, nb, BLOCK, dim).float() * ratio
    kv.copy_(values.to(E4M3).view(kv.shape))
    scales.copy_(scale.view(pages, nb, heads, 2).permute(0, 2, 3, 1))
    held = (rows / scale[block][..., None]).to(E4M3).permute(2, 0, 1, 3)
    kv.view(torch.uint8)[:, number, :, at % page] = held.transpose(0, 1).contiguous().view(
        torch.uint8)
    q = _norm_rope(st['q'], st['q_weight'], *args).to(dt)
    return q, _held(st)


def _attention(st):
    q, scales, table = st['q'], st['scales'], st['table'].long()
    _, _, hk, page, d = st['kv'].shape
    t, hq, _ = q.shape
    s, n = table.shape[0], st['max_new']
    g, keys = hq // hk, table.shape[1] * page
    starts, lengths = st['starts'].long(), st['lengths'].long()
    new = starts[1:] - starts[:-1]
    step = torch.arange(n, device='cuda')
    rows = (starts[:-1, None] + step).clamp(max=t - 1)
    queries = q[rows].float().view(s, n, hk, g, d).transpose(1, 2).reshape(s * hk, n * g, d)
    key = torch.arange(keys, device='cuda')
    seen = key < lengths[:, None]  # by some row
    k, v = (st['kv'][side].view(torch.uint8)[table].view(E4M3).float().view(
        *table.shape, hk, page // BLOCK, BLOCK, d) * scales[table, :, side][..., None, None]
        for side in range(2))
    k = k.transpose(1, 2).reshape(s * hk, keys, d)
    v = torch.where(seen[:, None, :, None], v.transpose(1, 2).reshape(s, hk, keys, d), 0.0)
    scores = torch.bmm(queries, k.transpose(1, 2)).mul_(d ** -0.5).view(s, hk, n, g, keys)
    behind = key <= (lengths - new)[:, None, None] + step[:, None]  # [s, n, keys]
    scores.masked_fill_(~(behind & seen[:, None])[:, None, :, None], float('-inf'))
    p = torch.exp(scores - scores.amax(-1, keepdim=True).clamp_min(-1e30))
    total = p.sum(-1, keepdim=True)
    o = torch.bmm(p.view(s * hk, n * g, keys), v.view(s * hk, keys, d)).view(s, hk, n, g, d)
    o = torch.where(total > 0, o / total, 0.0).transpose(1, 2).reshape(s, n, hq, d)
    seq, place, _ = _places(st)
    o = o[seq, place.clamp(max=n - 1)]
    if st['gate'] is not None:
        o = o / (1.0 + torch.exp(-st['gate'].float()))
    live = torch.arange(t, device='cuda') < starts[-1]
    return torch.where(live[:, None, None], o.to(q.dtype), st['out'])


def _norm_plain(st):
    h = st['h']
    h.copy_(h.float() + st['x'].float())
    v = h.float()
    v = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + st['eps']) * (1.0 + st['weight'])
    v = v.view(h.shape[0], -1, 128)
    s = v.abs().amax(-1, keepdim=True).clamp_min(1e-10) * (1.0 / 127.0)
    return torch.round(v / s).to(torch.int8).view(h.shape), s[..., 0]


def run(state):
    st = state
    if own:
        from localmoe35ba3b_amd.operators import attention, w8a8
        if st['kind'] == 'rotate':
            return attention.qk_norm_rope(st['q'], st['k'], st['q_weight'], st['k_weight'],
                                          st['positions'], st['inv_freq'], st['eps'],
                                          axes=st['axes'])
        if st['kind'] == 'append':
            axes = None if st['positions'] is None else st['axes']
            q = attention.append(st['kv'][0], st['kv'][1], st['k'], st['v'], st['starts'],
                                 st['lengths'], st['table'], inv_freq=st['inv_freq'],
                                 k_weight=st['k_weight'], q=st['q'], q_weight=st['q_weight'],
                                 eps=st['eps'], positions=st['positions'], axes=axes,
                                 scales=st['scales'])
            return q, _held(st)
        if st['kind'] == 'attention':
            return attention.paged_attention(st['q'], st['kv'][0], st['kv'][1], st['starts'],
                                             st['lengths'], st['table'], gate=st['gate'],
                                             max_new=st['max_new'], out=st['out'],
                                             scales=st['scales'])
        q, s = w8a8.norm_quantize(st['h'], st['weight'], st['eps'], add=st['x'])
    elif st['kind'] == 'rotate':
        args = st['positions'], st['axes'], st['inv_freq'], st['eps']
        return tuple(_norm_rope(st[n], st[n + '_weight'], *args).to(st['dtype']) for n in 'qk')
    elif st['kind'] == 'append':
        return _append_plain(st)
    elif st['kind'] == 'attention':
        return _attention(st)
    else:
        q, s = _norm_plain(st)
    return (q.view(*s.shape, 128) * s[..., None]).to(st['dtype']), st['h']


# ------------------------------------------------------------------ work
def work(case):
    if case['kind'] == 'norm':
        elements = case['tokens'] * case['hidden']
        # two rows read, one and its quarter (8 bits and a scale) written
        return dict(bytes=elements * 7 + elements // 32 + 4 * case['hidden'], flops=8 * elements)
    hq, hk, d, t = case['hq'], case['hk'], case['d'], _tokens(case)
    if case['kind'] == 'rotate':
        elements = t * (hq + hk) * d
        return dict(bytes=4 * elements + 8 * case['axes'] * t + 8 * d, flops=8 * elements)
    if case['kind'] == 'append':
        blocks = sum((l - 1) // BLOCK - (l - n) // BLOCK + 1 for n, l in _lengths(case))
        return dict(bytes=t * d * (4 * hq + 6 * hk) + 8 * hk * blocks + 8 * d,
                    flops=t * d * (8 * hq + 12 * hk))
    lengths = _lengths(case)
    rows = sum(n for n, _ in lengths)
    pairs = sum(n * (l - n) + n * (n + 1) // 2 for n, l in lengths)
    keys = sum(l for _, l in lengths)
    return dict(bytes=2 * d * (3 if case['gate'] else 2) * rows * hq + 2 * hk * keys * d
                + 2 * hk * keys // 4, flops=4 * hq * d * pairs)


# ------------------------------------------------------------------ 64-bit results
def _exact_rows(x, weight, positions, axes, inv_freq):
    """Pairs (i, i + half) of the normalized row as complex numbers, turned by the angle."""
    z = x.double()
    z = z / (z.square().sum(-1, keepdim=True) / z.shape[-1] + EPS).sqrt()
    z = z + z * weight.double()
    half = inv_freq.shape[0]
    angle = torch.stack([positions[a].double() * f for a, f in
                         zip(axes.tolist(), inv_freq.double().tolist())], -1)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device='cuda'), angle)
    pair = torch.complex(z[..., :half].contiguous(),
                         z[..., half:2 * half].contiguous()) * turn[:, None]
    z[..., :half], z[..., half:2 * half] = pair.real, pair.imag
    return z


def _exact_e4m3(z):
    """z rounded to four significant bits, or to multiples of 2^-9 below 2^-6."""
    power = torch.floor(torch.log2(z.abs().clamp_min(2.0 ** -6)))
    step = torch.exp2(power - 3)
    return torch.round(z / step) * step


def exact(case, seed):
    st = _inputs(case, seed)
    if case['kind'] == 'norm':
        h = (st['h'].double() + st['x'].double()).to(st['dtype']).double()
        n = h / (h.square().sum(-1, keepdim=True) / h.shape[-1] + EPS).sqrt()
        n = (n + n * st['weight'].double()).view(h.shape[0], -1, 128)
        s = n.abs().amax(-1, keepdim=True).clamp_min(1e-10) / 127
        return torch.round(n / s) * s, h
    if case['kind'] == 'rotate':
        return tuple(_exact_rows(st[n], st[n + '_weight'], st['positions'], st['axes'],
                                 st['inv_freq']) for n in ('q', 'k'))
    page, table, row = case['page'], st['table'].tolist(), 0
    held = st['kv'].double().view(2, -1, case['hk'], page // BLOCK, BLOCK, case['d'])
    held = (held * _blocks(st['scales']).double()).view(st['kv'].shape)
    if case['kind'] == 'append':
        dt, lengths = st['dtype'], _lengths(case)
        positions = st['positions']
        if positions is None:
            positions = torch.cat([torch.arange(l - n, l) for n, l in lengths])[None].to('cuda')
        args = positions, st['axes'], st['inv_freq']
        q = _exact_rows(st['q'], st['q_weight'], *args)
        sides = _exact_rows(st['k'], st['k_weight'], *args), st['v'].double()
        for s, (n, l) in enumerate(lengths):
            p = l - n
            while p < l:  # the part of one block
                m = min(BLOCK - p % BLOCK, l - p)
                number, at, b = table[s][p // page], p % page, p % page // BLOCK
                for side, rows in enumerate(sides):
                    x = rows[row:row + m].clamp(-MOST[dt], MOST[dt]).transpose(0, 1)
                    least = torch.exp2(torch.ceil(torch.log2(x.abs().amax((1, 2)) / 448)))
                    scale = least.clamp_min(2.0 ** LEAST[dt])
                    before = st['scales'][number, :, side, b].double()
                    if p % BLOCK:
                        scale = torch.maximum(scale, before)
                    behind = held[side, number, :, at + m:at + BLOCK - p % BLOCK]
                    behind *= (scale / before)[:, None, None]
                    scale = scale[:, None, None]
                    old = held[side, number, :, at - p % BLOCK:at]
                    old.copy_(_exact_e4m3(old / scale) * scale)
                    held[side, number, :, at:at + m] = _exact_e4m3(x / scale) * scale
                p, row = p + m, row + m
        return q, held
    out, g = st['out'].double(), case['hq'] // case['hk']
    for s, (n, l) in enumerate(_lengths(case)):
        used = table[s][:-(-l // page)]
        for h in range(case['hk']):
            k, v = (held[side, used, h].reshape(-1, case['d'])[:l] for side in range(2))
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
