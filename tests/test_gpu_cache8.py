"""GPU tests of the cache in 8 bits against 64-bit results: the append with its scales, attention
over it, rotation by positions of several axes, and the three run together."""
import math

import pytest
import torch

from localmoe35ba3b_amd.operators import attention as A
from tests import attention_util as U
from tests import cache8_util as C
from tests.conftest import seeded
from tests.test_gpu_attention import CHUNKS, DECODE, rand, to
from tests.test_gpu_attention import attend as attend16

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16
TYPES = pytest.mark.parametrize('dtype', [BF16, FP16])
I32 = torch.int32


def ints(*v):
    return torch.tensor(v, dtype=I32)


# ------------------------------------------------------------------ positions of several axes
@TYPES
@pytest.mark.parametrize('tokens,q_heads,k_heads,dim,pairs,axes', [
    (1, 16, 2, 256, 32, 3), (5, 3, 1, 256, 128, 2), (37, 32, 8, 128, 64, 3), (6, 1, 1, 64, 8, 1),
    (130, 7, 5, 64, 24, 4)])
def test_rotation_by_axes(dev, tokens, q_heads, k_heads, dim, pairs, axes, dtype):
    gen = seeded(tokens + dim)
    q, k = rand(gen, tokens, q_heads, dim, dtype=dtype), rand(gen, tokens, k_heads, dim, dtype=dtype)
    qw, kw = torch.randn(dim, generator=gen) * 0.2, torch.randn(dim, generator=gen) * 0.2
    positions = torch.randint(-(1 << 10), 1 << 20, (axes, tokens), generator=gen)
    axis = torch.randint(0, axes, (pairs,), generator=gen)
    freq = U.frequencies(pairs)
    args = to(dev, q, k, qw, kw)
    got = A.qk_norm_rope(*args, *to(dev, positions, freq), axes=axis.to(dev, I32))
    # a pair's angle by its axis: the oracle's rotation with a position for each pair
    for g, x, w, what in zip(got, (q, k), (qw, kw), 'qk'):
        parts = [U.norm_rope(x, w, positions[a], freq) for a in range(axes)]
        want, slack = parts[0][0].clone(), parts[0][1]
        for i, a in enumerate(axis.tolist()):
            want[..., [i, i + pairs]] = parts[a][0][..., [i, i + pairs]]
        U.assert_rows(g, want, slack, dtype, what)


def test_axes_of_other_types_and_out_of_range(dev):
    """int32 positions with a stride, int64 axes beyond the last (taken as the last), and one axis
    alone, which is what plain positions are."""
    gen = seeded(3)
    q, k, freq = rand(gen, 9, 2, 64), rand(gen, 9, 1, 64), U.frequencies(16)
    positions = torch.randint(0, 5000, (9, 3), generator=gen)
    axis = torch.tensor([0, 1, 2, 9, -4] + [1] * 11)
    args = to(dev, q, k, None, None)
    fd, pd = to(dev, freq, positions)
    a = A.qk_norm_rope(*args, pd.int().t(), fd, axes=axis.to(dev))
    b = A.qk_norm_rope(*args, pd.t().contiguous(), fd, axes=axis.clamp(0, 2).to(dev, I32))
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    one = A.qk_norm_rope(*args, pd[:, 1].contiguous()[None], fd, axes=axis.to(dev))
    plain = A.qk_norm_rope(*args, pd[:, 1].contiguous(), fd)
    assert all(torch.equal(x, y) for x, y in zip(one, plain))


@pytest.mark.parametrize('eight', [False, True])
def test_append_by_positions(dev, eight):
    """Positions count for the rotation, places for the cache: what qk_norm_rope gives for them is
    what the append holds, and the queries' rows are the same bits."""
    gen, dim, pairs = seeded(5), 128, 24
    lens = [(5, 40), (1, 3), (20, 20), (0, 7)]
    starts, lengths, table, pages = U.batch(lens, 16)
    n = int(starts[-1]) + 2
    q, k, v = rand(gen, n, 4, dim), rand(gen, n, 2, dim), rand(gen, n, 2, dim)
    weights = torch.randn(dim, generator=gen) * 0.1
    positions = torch.randint(0, 9000, (3, n), generator=gen)
    axis, freq = torch.arange(pairs, dtype=I32) % 3, U.frequencies(pairs)
    qd, kd, vd, wd, pd, ad, fd = to(dev, q, k, v, weights, positions, axis, freq)
    batch = to(dev, starts, lengths, table)
    if eight:
        kp, vp, scales = to(dev, *C.random_cache(gen, pages, 2, 16, dim, BF16))
    else:
        kp, vp, scales = *to(dev, *(rand(gen, pages, 2, 16, dim) for _ in range(2))), None
    got = A.append(kp, vp, kd, vd, *batch, inv_freq=fd, k_weight=wd, q=qd, q_weight=wd,
                   positions=pd, axes=ad, scales=scales)
    wq, wk = A.qk_norm_rope(qd, kd, wd, wd, pd, fd, axes=ad)
    assert torch.equal(got[:-2], wq[:-2]) and not got[-2:].any()
    for p, axes in ((pd[1], None), (pd[1:2], ad)):  # one axis, either way
        again = A.append(kp.clone(), vp.clone(), kd, vd, *batch, inv_freq=fd, k_weight=wd, q=qd,
                         q_weight=wd, positions=p, axes=axes, scales=scales)
        assert torch.equal(again[:-2], A.qk_norm_rope(qd, kd, wd, wd, pd[1], fd)[0][:-2])
    values = C.held(kp, vp, scales)[0] if eight else kp.cpu().double()
    for s, (new, length) in enumerate(lens):
        for i in range(new):
            p, row = length - new + i, int(starts[s]) + i
            x = values[int(table[s, p // 16]), :, p % 16]
            want = wk[row].cpu().double()
            if eight:  # a rounding to bf16 and one to e4m3, of blocks at least as large as the row
                top = want.abs().amax(-1, keepdim=True)
                assert ((x - want).abs() <= 2.0 ** -4 * 1.01 * want.abs() + 2.0 ** -7 * top).all()
            else:
                assert torch.equal(x, want)


# ------------------------------------------------------------------ append
def run_append(dev, calls, page, heads, dim, dtype, q_heads=3, pairs=16, seed=0, strange=False):
    """calls: lists of (sequence, new tokens) appended one after another to sequences that begin
    empty, in pages that hold anything; values bit for bit, keys within their roundings."""
    gen = seeded(seed)
    count = 1 + max(s for call in calls for s, _ in call)
    total = [sum(n for call in calls for t, n in call if t == s) for s in range(count)]
    _, _, table, pages = U.batch([(0, n) for n in total], page, seed)
    kp, vp, scales = to(dev, *C.random_cache(gen, pages, heads, page, dim, dtype))
    want = [x.clone() for x in C.held(kp, vp, scales)]
    scale64 = scales.cpu().double()
    kw, qw, freq = torch.randn(dim, generator=gen) * 0.2, torch.zeros(dim), U.frequencies(pairs)
    length = [0] * count
    for call in calls:
        n = sum(m for _, m in call)
        sizes = torch.exp2(torch.randint(-9, 9, (n, 1, 1), generator=gen).float())
        q, k = rand(gen, n, q_heads, dim, dtype=dtype), rand(gen, n, heads, dim, dtype=dtype)
        v = (torch.randn(n, heads, dim, generator=gen) * sizes).to(dtype)
        k[:, :, 0] *= 3.0
        if strange:  # zeros, values beyond the type's four bits, and what is not finite
            v[0, 0], v[-1, -1, :3] = 0, torch.tensor([math.inf, math.nan, -math.inf])
            v[n // 2, 0, 5] = torch.finfo(dtype).max
            v[n // 2, -1, 7] = -torch.finfo(dtype).tiny
        new = [m for _, m in call]
        for s, m in call:
            length[s] += m
        starts = torch.tensor([0] + new).cumsum(0).to(I32)
        rows = torch.tensor([s for s, _ in call])
        lengths = torch.tensor([length[s] for s, _ in call], dtype=I32)
        got = A.append(kp, vp, *to(dev, k, v, starts, lengths, table[rows]),
                       inv_freq=freq.to(dev), k_weight=kw.to(dev), q=q.to(dev), q_weight=qw.to(dev),
                       scales=scales)
        for (s, m), at in zip(call, starts.tolist()):
            base = length[s] - m
            positions = torch.arange(base, base + m)
            k64, slack = U.norm_rope(k[at:at + m], kw, positions, freq)
            U.assert_rows(got[at:at + m], *U.norm_rope(q[at:at + m], qw, positions, freq), dtype, 'q')
            args = base, table[s].tolist(), page, dtype
            C.append(want[1], scale64[:, :, 1], v[at:at + m].double(), *args)
            now = C.held(kp, vp, scales)
            used = C.append(want[0], scale64[:, :, 0], k64, *args)
            for i, p in enumerate(range(base, base + m)):
                number, b = int(table[s, p // page]), p % page // C.BLOCK
                x = now[0][number, :, p % page]
                theirs = scales[number, :, 0, b].cpu().double()[:, None]
                # a scale of twice or half the oracle's only where the largest value is at a border
                assert ((theirs / used[i][:, None] - 1).abs() < 1.01).all()
                C.assert_keys(x, k64[i], slack[i], torch.maximum(theirs, used[i][:, None]),
                              f'keys {s} {p}')
        # what the kernel holds is what the next call starts from
        want[0], scale64[:, :, 0] = now[0].clone(), scales[:, :, 0].cpu().double()
        assert torch.equal(scales[:, :, 1].cpu().double(), scale64[:, :, 1]), 'scales of values'
        assert torch.equal(now[1].nan_to_num(-1.0), want[1].nan_to_num(-1.0)), 'values'
        assert torch.equal(now[1].isnan(), want[1].isnan())
    return kp, vp, scales, table, length


@TYPES
@pytest.mark.parametrize('dim,heads', [(64, 1), (64, 5), (128, 2), (256, 2), (256, 9)])
def test_append_whole_and_parts(dev, dim, heads, dtype):
    """A prompt that ends inside a block, one token, a chunk over several pages, a whole block."""
    run_append(dev, [[(0, 37)], [(0, 1)], [(0, 50)], [(0, 8)], [(0, 16)]], 32, heads, dim, dtype,
               seed=dim)


@TYPES
@pytest.mark.parametrize('page', [16, 64])
def test_append_tokens_that_grow_a_block(dev, page, dtype):
    """Token by token: a block's scale grows with its rows, which are rounded again."""
    run_append(dev, [[(0, 1)]] * 20 + [[(0, 3)]] * 4, page, 2, 64, dtype, seed=page)


@TYPES
def test_append_several_sequences(dev, dtype):
    run_append(dev, [[(0, 5), (1, 33), (2, 1)], [(1, 1), (0, 1), (2, 40)], [(2, 1), (1, 16)]], 16, 2,
               128, dtype, seed=3)


@TYPES
def test_append_strange_values(dev, dtype):
    run_append(dev, [[(0, 9)], [(0, 9)], [(0, 1)], [(0, 30)]], 16, 2, 64, dtype, seed=7, strange=True)


@pytest.mark.parametrize('sequences', [64, 65, 300])
def test_append_many_sequences(dev, sequences):
    """More sequences than a wave or a workgroup looks at together, some without a new token."""
    first = [(s, s % 5) for s in range(sequences)]
    run_append(dev, [first, [(s, 1) for s in range(sequences)]], 16, 1, 64, BF16, seed=sequences)


@TYPES
def test_append_after_positions_are_taken_back(dev, dtype):
    """A draft whose last tokens are dropped: the block keeps its scale, and the dropped rows' bits
    where no new row comes; from the block's begin on, the scale is the new rows'."""
    gen = seeded(5)
    kp, vp, scales = to(dev, *C.random_cache(gen, 3, 2, 16, 64, dtype))
    want, scale64 = C.held(kp, vp, scales)[1], scales[:, :, 1].cpu().double()
    table = [2, 0]
    for base, n, size in ((0, 30, 1.0), (30, 2, 900.0), (20, 3, 1.0), (16, 5, 0.25), (3, 1, 40.0)):
        v = rand(gen, n, 2, 64, dtype=dtype) * size
        A.append(kp, vp, *to(dev, v, v, ints(0, n), ints(base + n), ints(*table).view(1, 2)),
                 scales=scales)
        C.append(want, scale64, v.double(), base, table, 16, dtype)
        assert torch.equal(C.held(kp, vp, scales)[1], want), (base, n)
        assert torch.equal(scales[:, :, 1].cpu().double(), scale64), (base, n)


def test_append_outside_the_table(dev):
    """Positions before 0 or behind the table's pages, and page numbers out of range; rows of no
    sequence leave the cache as it is."""
    v = rand(seeded(2), 10, 1, 64)
    kp = torch.zeros(3, 1, 16, 64, device=dev).to(C.E4M3)
    scales = torch.ones(3, 1, 2, 1, device=dev)
    vp = kp.clone()
    table = torch.tensor([[0, 1], [2, 99]], dtype=I32)  # 99 is taken as the last page
    lengths = ints(2, 34)  # positions -2 .. 1 and 30 .. 33
    q = A.append(kp, vp, *to(dev, v, v, ints(0, 4, 8), lengths, table), q=v.to(dev), scales=scales)
    assert not q[8:].any()
    rows = v.double()
    want = torch.zeros(3, 1, 16, 64, dtype=torch.float64)
    w = torch.ones(3, 1, 1, dtype=torch.float64)
    C.append(want, w, rows[2:4], 0, [0, 1], 16, BF16)
    C.append(want, w, rows[4:6], 14, [2, 2], 16, BF16)
    assert torch.equal(C.held(kp, vp, scales)[1], want)
    assert torch.equal(scales[:, :, 1].cpu().double(), w)


def test_append_without_sequences(dev):
    kp, vp, scales = to(dev, *C.random_cache(seeded(1), 4, 2, 16, 64, BF16))
    before = kp.clone(), scales.clone()
    q, k = rand(seeded(2), 5, 4, 64).to(dev), rand(seeded(3), 5, 2, 64).to(dev)
    none = torch.zeros(1, dtype=I32, device=dev)
    got = A.append(kp, vp, k, k, none, none[:0], none[:0].view(0, 1), q=q, scales=scales)
    assert not got.any() and torch.equal(kp.view(torch.uint8), before[0].view(torch.uint8))
    assert torch.equal(scales, before[1])
    batch = to(dev, ints(0, 0), ints(9), ints(0).view(1, 1))  # a sequence without a new token
    assert not A.append(kp, vp, k, k, *batch, q=q, scales=scales).any()
    assert torch.equal(scales, before[1])


# ------------------------------------------------------------------ attention
def attend(dev, lens, page, q_heads, heads, dim, dtype, gate=False, pad=0, seed=0, scale=None,
           max_new=None, sharp=1.0, spread=3.0):
    gen = seeded(seed)
    starts, lengths, table, pages = U.batch(lens, page, seed)
    tokens = int(starts[-1]) + pad
    q = rand(gen, tokens, q_heads, dim, dtype=dtype, scale=sharp)
    g = rand(gen, tokens, q_heads, dim, dtype=dtype) if gate else None
    kp, vp, scales = C.random_cache(gen, pages, heads, page, dim, dtype, spread)
    k64, v64 = C.held(kp, vp, scales, dtype)
    # what no sequence holds must not matter, whatever it is: NaN in the rows and scales of any bits
    used = torch.zeros(pages, page, dtype=torch.bool)
    for s, (_, n) in enumerate(lens):
        for p in range(n):
            used[int(table[s, p // page]), p % page] = True
    sides = [x.transpose(1, 2).clone().view(torch.uint8) for x in (kp, vp)]
    for x in sides:
        x[~used] = 0x7F
    blocks = used.view(pages, -1, C.BLOCK).any(-1)
    odd = torch.tensor([math.inf, math.nan, 0.0, -math.inf])
    scales.transpose(1, 3)[~blocks] = odd[:2].view(1, 2, 1)
    kd, vd = (x.view(C.E4M3).transpose(1, 2).contiguous().to(dev) for x in sides)
    before = torch.full(q.shape, 7.0, dtype=dtype, device=dev)
    out = before.clone()
    args = to(dev, q, kd, vd, starts, lengths, table)
    got = A.paged_attention(*args, scale=scale, gate=to(dev, g)[0], max_new=max_new, out=out,
                            scales=scales.to(dev))
    assert got is out
    U.assert_attention(got, U.attention(q, k64, v64, starts, lengths, table, scale, g),
                       f'{lens} {page} {q_heads}/{heads} {dim}', before)


@TYPES
@pytest.mark.parametrize('lens,page,q_heads,heads,dim', DECODE)
def test_attention_few_tokens(dev, lens, page, q_heads, heads, dim, dtype):
    attend(dev, lens, page, q_heads, heads, dim, dtype, seed=dim, max_new=max(c for c, _ in lens))


@TYPES
@pytest.mark.parametrize('gate', [False, True])
@pytest.mark.parametrize('lens,page,q_heads,heads,dim', CHUNKS)
def test_attention_chunks(dev, lens, page, q_heads, heads, dim, gate, dtype):
    attend(dev, lens, page, q_heads, heads, dim, dtype, gate, pad=3, seed=dim)


@TYPES
@pytest.mark.parametrize('sharp', [1e-3, 8.0, 60.0])
def test_attention_flat_and_sharp_scores(dev, sharp, dtype):
    attend(dev, [(1, 700), (60, 400)], 16, 8, 2, 128, dtype, sharp=sharp, scale=0.11)


@pytest.mark.parametrize('dim', [64, 128, 256])
def test_attention_every_length(dev, dim):
    """Lengths around the steps, blocks and tiles, for one token and for chunks."""
    edges = [1, 15, 16, 17, 31, 32, 33, 47, 63, 64, 65, 95, 96, 97, 127, 128, 129, 160, 255, 256, 257]
    attend(dev, [(1, n) for n in edges], 16, 4, 2, dim, BF16, seed=dim, max_new=1)
    attend(dev, [(min(n, 40), n) for n in edges], 16, 4, 2, dim, BF16, seed=dim + 1)


def test_attention_negative_and_zero_scale(dev):
    for scale in (0.0, -0.2):
        attend(dev, [(1, 90), (20, 130)], 16, 4, 2, 64, BF16, scale=scale)


@pytest.mark.parametrize('sequences', [70, 300])
@pytest.mark.parametrize('chunks', [False, True])
def test_attention_many_sequences(dev, sequences, chunks):
    gen = torch.Generator().manual_seed(sequences)
    length = torch.randint(0, 90, (sequences,), generator=gen).tolist()
    lens = [(i % 4 if i % 7 else 30 * chunks, n) for i, n in enumerate(length)]
    lens = [(new, max(n, new - 1)) for new, n in lens]
    attend(dev, lens, 16, 4, 2, 64, BF16, gate=chunks, pad=2, seed=sequences,
           max_new=max(n for n, _ in lens))


@pytest.mark.parametrize('dim', [64, 128, 256])
@pytest.mark.parametrize('sequences,tokens,prompts', [(9, 3, 3), (40, 30, 0), (40, 0, 11), (70, 30, 9),
                                                      (300, 90, 5)])
def test_attention_tokens_beside_prompts(dev, sequences, tokens, prompts, dim):
    """Single tokens and prompts of one call, behind many keys and none, among sequences that have no
    new token; also where a call could have both and has one kind alone."""
    gen = torch.Generator().manual_seed(sequences)
    kind = torch.randperm(sequences, generator=gen).tolist()
    lens = []
    for i in kind:
        new = 1 if i < tokens else 20 + i * 37 % 150 if i < tokens + prompts else 0
        lens.append((new, new + i * 131 % (1200 if sequences < 100 else 300)))
    for call in (attend, attend16):
        call(dev, lens, 16, 8, 2, dim, BF16, gate=True, pad=2, seed=dim)


@pytest.mark.parametrize('new,heads,keys,dim', [(2, 128, 36000, 64), (2, 128, 20000, 128),
                                                (1, 128, 20000, 256), (20, 128, 10000, 64),
                                                (20, 128, 6000, 128), (20, 128, 4700, 256)])
def test_attention_long_parts(dev, new, heads, keys, dim):
    """Parts of a sequence longer than the pages and scales that a wave looks up at a time."""
    gen = torch.Generator(device=dev)
    gen.manual_seed(keys)
    pages = -(-keys // 64)
    kp, vp = ((torch.randn(pages, heads, 64, dim, generator=gen, device=dev) * 64).clamp_(-448, 448)
              .to(C.E4M3) for _ in range(2))
    scales = torch.exp2(torch.randint(-9, -3, (pages, heads, 2, 4), generator=gen, device=dev).float())
    table = torch.randperm(pages, generator=seeded(keys)).to(I32)[None]
    q = rand(seeded(keys), new, heads, dim)
    batch = ints(0, new), ints(keys), table
    got = A.paged_attention(q.to(dev), kp, vp, *to(dev, *batch), scales=scales)
    some = [0, heads // 2, heads - 1]  # heads are independent: three of them in 64 bits
    k, v = C.held(kp.view(torch.uint8)[:, some].view(C.E4M3), vp.view(torch.uint8)[:, some].view(C.E4M3),
                  scales[:, some], BF16)
    U.assert_attention(got[:, some], U.attention(q[:, some], k, v, *batch), f'{new} {keys} {dim}')
    assert got.isfinite().all()


@TYPES
@pytest.mark.parametrize('dim', [64, 128, 256])
@pytest.mark.parametrize('new', [1, 40])
def test_attention_odd_values(dev, new, dim, dtype):
    """NaN among the keys and values of a position that only the last rows see, and a scale beyond
    the type behind it: they show in those rows and in no other."""
    lens = [(new, 100), (new, 70)]
    gen = seeded(dim + new)
    starts, lengths, table, pages = U.batch(lens, 16)
    q = rand(gen, 2 * new, 4, dim, dtype=dtype)
    kp, vp, scales = C.random_cache(gen, pages, 2, 16, dim, dtype)
    clean = U.attention(q, *C.held(kp, vp, scales, dtype), starts, lengths, table)
    bad = 100 - max(1, new // 2)
    at = int(table[0, bad // 16])
    kb, vb = kp.view(torch.uint8), vp.view(torch.uint8)
    vb[at, 0, bad % 16, 3], vb[at, 0, bad % 16, dim - 2], kb[at, 1, bad % 16, 9] = 0x7F, 0xFF, 0x7F
    got = A.paged_attention(*to(dev, q, kp, vp, starts, lengths, table), scales=scales.to(dev)).cpu()
    sees = torch.zeros(2 * new, 4, dim, dtype=torch.bool)
    rows = slice(max(0, new - (100 - bad)), new)
    sees[rows, :2, 3] = sees[rows, :2, dim - 2] = True
    sees[rows, 2:] = True
    assert not got[sees].isfinite().any()
    U.assert_rows(got[~sees], clean[0][~sees], clean[1][~sees], dtype, 'rows before it')


@TYPES
@pytest.mark.parametrize('new', [1, 30])
def test_attention_every_code_and_scale(dev, new, dtype):
    """All 254 values under scales from the least to the largest that the append makes: with equal
    weights a result is the mean of the values, so each must be exact."""
    dim, heads, page = 64, 6, 16
    codes = torch.tensor([c for c in range(256) if c & 0x7F != 0x7F], dtype=torch.uint8)
    codes = torch.cat([codes, codes[:2]]).view(4, dim)  # four rows
    vp = codes[torch.arange(page) % 4].view(1, 1, page, dim).expand(2, heads, page, dim).contiguous()
    exps = [-100, -60, -1, 0, 50, 100] if dtype == BF16 else [-15, -9, -1, 0, 3, 7]
    scales = torch.exp2(torch.tensor(exps).float()).view(1, heads, 1, 1).expand(2, heads, 2, 1).contiguous()
    kp = torch.zeros(2, heads, page, dim).to(C.E4M3)
    starts, lengths = ints(0, new), ints(new - 1 + 4)
    q = torch.zeros(new, heads, dim, dtype=dtype)
    kv = C.held(kp, vp.view(C.E4M3), scales, dtype)
    assert all(x.isfinite().all() for x in kv)
    table = ints(0, 1, 0).view(1, 3)
    got = A.paged_attention(*to(dev, q, kp, vp.view(C.E4M3), starts, lengths, table),
                            scales=scales.to(dev))
    U.assert_attention(got, U.attention(q, *kv, starts, lengths, table), 'codes')


@TYPES
@pytest.mark.parametrize('dim', [64, 128, 256])
@pytest.mark.parametrize('new', [1, 40])
def test_attention_values_beyond_the_type_that_no_row_sees(dev, new, dim, dtype):
    """Under the largest scale the upper 8-bit values are infinities of the type: behind a sequence's
    end they reach no row, and before it only those that see them."""
    gen = seeded(dim)
    lens = [(new, 85), (new, 70)]
    starts, lengths, table, pages = U.batch(lens, 16)
    q = rand(gen, 2 * new, 4, dim, dtype=dtype)
    kp, vp, scales = C.random_cache(gen, pages, 2, 16, dim, dtype)
    last = [int(table[s, n // 16]) for s, (_, n) in enumerate(lens)]  # blocks that rows go on in
    scales[last, :, 1] = 2.0 ** (120 if dtype == BF16 else 8)
    vb = vp.view(torch.uint8)
    for at, (_, n) in zip(last, lens):
        vb[at] = torch.randint(0, 2, vb[at].shape, generator=gen).to(torch.uint8)  # tiny, seen
        vb[at, :, n % 16:] = torch.randint(0x78, 0x7F, vb[at, :, n % 16:].shape, generator=gen).to(torch.uint8)
    k64, v64 = C.held(kp, vp, scales, dtype)
    for at, (_, n) in zip(last, lens):
        assert v64[at, :, n % 16:].isinf().all()
    got = A.paged_attention(*to(dev, q, kp, vp, starts, lengths, table), scales=scales.to(dev)).cpu()
    want = U.attention(q, k64, v64, starts, lengths, table)
    U.assert_attention(got, want, 'behind the end')
    at, bad = last[0], 85 - max(1, new // 2)  # a position of sequence 0 that its last rows see
    if bad // 16 == 85 // 16:
        vb[at, 0, bad % 16, 3] = 0x78
        got = A.paged_attention(*to(dev, q, kp, vp, starts, lengths, table), scales=scales.to(dev)).cpu()
        assert got[new - (85 - bad):new, :2, 3].isinf().all()
        got[new - (85 - bad):new, :2, 3] = want[0][new - (85 - bad):new, :2, 3].to(dtype)
        U.assert_attention(got, want, 'rows before it')


def test_attention_malformed_batches_stay_in_bounds(dev):
    """Page numbers, lengths and starts out of range, for both operators: some result, no access
    outside."""
    q, k = to(dev, rand(seeded(1), 40, 4, 64), rand(seeded(2), 40, 2, 64))
    kp, vp, scales = to(dev, *C.random_cache(seeded(3), 5, 2, 16, 64, BF16))
    on = lambda *v: ints(*v).to(dev)
    table = torch.stack([on(0, 99, -3), on(1, 2, 2 ** 31 - 1)])
    for starts, lengths in ((on(0, 20, 40), on(1000, -5)), (on(0, 30, 100), on(48, 48)),
                            (on(-9, 20, 10), on(48, 40)), (on(50, 60, 70), on(4, 4)),
                            (on(0, 1, 2), on(2 ** 31 - 1, -2 ** 31))):
        A.append(kp, vp, k, k, starts, lengths, table, q=q, scales=scales)
        for max_new in (1, 40):
            A.paged_attention(q, kp, vp, starts, lengths, table, max_new=max_new, scales=scales)
            torch.cuda.synchronize()


def test_layouts(dev):
    """Pages and scales of one layer of a cache that holds several, strided queries, one shared
    table."""
    gen, page, dim, heads = seeded(9), 32, 128, 2
    lens = [(1, 90), (1, 90), (1, 90)]
    kp, vp, scales = C.random_cache(gen, 6, heads, page, dim, BF16)
    kv = torch.stack([kp.view(torch.uint8), vp.view(torch.uint8)], 1)  # [pages, 2, ...]
    three = scales[:, None].expand(6, 3, heads, 2, 2).contiguous()
    row = torch.randperm(6, generator=gen)[:3].to(I32)
    starts, lengths = ints(0, 1, 2, 3), ints(90, 50, 1)
    qg = rand(gen, 8, 3, 2 * dim).transpose(0, 1)
    kvd, sd, rd, qd, st, ld = to(dev, kv, three, row, qg, starts, lengths)
    kvd = kvd.view(C.E4M3)
    got = A.paged_attention(qd[..., :dim], kvd[:, 0], kvd[:, 1], st, ld, rd.expand(3, 3),
                            gate=qd[..., dim:], max_new=1, scales=sd[:, 1])
    want = U.attention(qg[..., :dim], *C.held(kp, vp, scales, BF16), starts, lengths,
                       row.expand(3, 3), gate=qg[..., dim:])
    U.assert_attention(got, want, 'strided')
    k = rand(gen, 3, heads, dim).to(dev)
    own = torch.tensor([[0, 1, 2], [3, 4, 5], [3, 4, 5]], dtype=I32, device=dev)[:2]
    plain = kvd[:, 0].clone(), kvd[:, 1].clone(), sd[:, 1].clone()
    for c in ((kvd[:, 0], kvd[:, 1], sd[:, 1]), plain):
        A.append(c[0], c[1], k, k, *to(dev, ints(0, 1, 3), ints(90, 41)), own, scales=c[2])
    for a, b in zip((kvd[:, 0], kvd[:, 1]), plain):
        assert torch.equal(a.contiguous().view(torch.uint8), b.view(torch.uint8))
    assert torch.equal(sd[:, 1], plain[2])


def test_far_pages(dev):
    """Offsets beyond 32 bits: 4.3 GB of keys, of which a sequence's pages lie at the end."""
    heads, page, dim, n = 2, 1024, 256, 1500
    pages = (1 << 32) // (heads * page * dim) + 3
    kd = torch.empty(pages, heads, page, dim, dtype=C.E4M3, device=dev)
    vd = torch.empty(pages, heads, page, dim, dtype=C.E4M3, device=dev)
    sd = torch.ones(pages, heads, 2, page // 16, device=dev)
    gen = seeded(10)
    k, v, s = C.random_cache(gen, 2, heads, page, dim, BF16)
    kd[-2:], vd[-2:], sd[-2:] = to(dev, k, v, s)
    starts, lengths = ints(0, 1, 30), ints(n, n)
    q = rand(gen, 30, 4, dim)
    table = torch.tensor([[0, 1], [1, 0]], dtype=I32)
    far = (table + pages - 2).to(dev)
    got = A.paged_attention(*to(dev, q), kd, vd, *to(dev, starts, lengths), far, scales=sd)
    U.assert_attention(got, U.attention(q, *C.held(k, v, s, BF16), starts, lengths, table), 'far')
    new = rand(gen, 2, heads, dim)
    A.append(kd, vd, *to(dev, new, new, ints(0, 1, 2), lengths), far, scales=sd)
    for row, number in ((0, -1), (1, -2)):
        scale = sd[number, :, 1, (n - 1) % page // 16].cpu().double()[:, None]
        x = vd[number, :, (n - 1) % page].cpu().double() * scale
        assert torch.equal(x, C.e4m3(new[row].double() / scale) * scale)


# ------------------------------------------------------------------ together
def step(cache, scales, q, k, v, gate, qw, kw, freq, batch, max_new, positions=None, axes=None):
    q = A.append(*cache, k, v, *batch, inv_freq=freq, k_weight=kw, q=q, q_weight=qw,
                 positions=positions, axes=axes, scales=scales)
    return A.paged_attention(q, *cache, *batch, gate=gate, max_new=max_new, scales=scales)


@TYPES
def test_prompt_in_chunks_then_tokens(dev, dtype):
    """A prompt with an image in ragged chunks, then tokens, against attention in 64 bits over what
    the cache holds in the end.  Blocks that later calls went on with were rounded again only below
    2^-6 of their scale, which the tolerance counts: a key's products with |q| and a value's weight."""
    gen, dim, hq, hk, page, total = seeded(11), 128, 6, 2, 16, 96
    q, k, v, gate = (rand(gen, total, h, dim, dtype=dtype) for h in (hq, hk, hk, hq))
    qw, kw, freq = torch.randn(dim, generator=gen) * 0.1, torch.randn(dim, generator=gen) * 0.1, \
        U.frequencies(32)
    positions = torch.stack([torch.arange(total), torch.arange(total) // 5, torch.arange(total) % 5])
    axes = (torch.arange(32) % 3).to(I32).to(dev)
    kp, vp, scales = to(dev, *C.random_cache(gen, 8, hk, page, dim, dtype))
    table = torch.tensor([[5, 0, 7, 1, 3, 2]], dtype=I32, device=dev)
    weights = to(dev, qw, kw, freq)
    for counts in ((32, 16, 48), (37, 1, 2, 46, 1, 1, 1, 1, 6)):
        at, seen = 0, []
        for count in counts:
            rows = slice(at, at + count)
            at += count
            batch = *to(dev, ints(0, count), ints(at)), table
            p = positions[:, rows].contiguous().to(dev)
            got = step((kp, vp), scales, *to(dev, q[rows], k[rows], v[rows], gate[rows]), *weights,
                       batch, count, p, axes)
            # against what the cache holds right after the call
            qs, _ = A.qk_norm_rope(*to(dev, q[rows], k[rows], qw, kw), p, weights[2], axes=axes)
            want = U.attention(qs.cpu(), *C.held(kp, vp, scales, dtype), ints(0, count), ints(at),
                               table.cpu(), gate=gate[rows])
            U.assert_attention(got, want, f'{counts} at {at}')


def test_captured_step_follows_its_batch(dev):
    """A captured decode step replayed while lengths, positions and inputs change between replays,
    with eager work in between; two graphs alive at once."""
    gen, dim, hq, hk, page = seeded(12), 256, 16, 2, 16
    kp, vp, scales = to(dev, *C.random_cache(gen, 40, hk, page, dim, BF16))
    starts, lengths = to(dev, ints(0, 1, 2, 3), ints(5, 170, 33))
    table = torch.randperm(40, generator=gen)[:36].view(3, 12).to(dev, I32)
    positions = torch.tensor([[5, 170, 33], [2, 90, 11]], device=dev)
    axes = (torch.arange(32) % 2).to(dev, I32)
    ins = [rand(gen, 3, h, dim).to(dev) for h in (hq, hk, hk, hq)]
    weights = to(dev, torch.zeros(dim), torch.zeros(dim), U.frequencies(32))
    run = lambda c, s: step(c, s, *ins, *weights, (starts, lengths, table), 1, positions, axes)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run((kp, vp), scales)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run((kp, vp), scales)
        graphs.append((graph, out))
    for i in range(6):
        lengths += 1
        positions += 1
        for x in ins:
            x.copy_(rand(gen, *x.shape) * 2.0 ** (i % 3))
        eager, eager_scales = [kp.clone(), vp.clone()], scales.clone()
        graph, out = graphs[i % 2]
        graph.replay()
        want = run(eager, eager_scales)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(scales, eager_scales)
        for a, b in zip((kp, vp), eager):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize('eight', [False, True])
@pytest.mark.parametrize('dim', [64, 128, 256])
def test_captured_call_of_any_kind(dev, dim, eight):
    """One captured call, replayed for prompts beside single tokens, one kind alone and no new token at
    all: what the batch then holds decides, bit for bit as in a call of its own."""
    gen, tokens, page = seeded(dim), 150, 16
    kp, vp, scales = C.random_cache(gen, 500, 2, page, dim, BF16)
    if not eight:
        kp, vp = rand(gen, 500, 2, page, dim), rand(gen, 500, 2, page, dim)
    kp, vp, q, gate = to(dev, kp, vp, rand(gen, tokens, 8, dim), rand(gen, tokens, 8, dim))
    scales = scales.to(dev) if eight else None
    table = torch.randperm(500, generator=gen)[:480].view(12, 40).to(I32).to(dev)
    kinds = [[(1, 600 - 40 * i) for i in range(9)] + [(70, 100), (30, 500), (9, 9)],
             [(1, 50 * i + 1) for i in range(12)], [(0, 7)] * 12,
             [(40, 640), (0, 0), (50, 60)] + [(0, 3)] * 8 + [(60, 300)],
             [(0, 0)] * 4 + [(2, 640)] * 4 + [(30, 31)] + [(1, 1)] * 3]
    starts, lengths = torch.zeros(13, dtype=I32, device=dev), torch.zeros(12, dtype=I32, device=dev)
    out = torch.zeros_like(q)

    def call(o):
        return A.paged_attention(q, kp, vp, starts, lengths, table, gate=gate, out=o, scales=scales)

    call(out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out)
    for lens in kinds + kinds[::-1]:
        starts.copy_(torch.tensor([0] + [n for n, _ in lens]).cumsum(0))
        lengths.copy_(torch.tensor([n for _, n in lens]))
        out.fill_(3.0)
        graph.replay()
        want = call(torch.full_like(q, 3.0))
        torch.cuda.synchronize()
        assert torch.equal(out, want), lens
        assert (out[int(starts[-1]):] == 3.0).all()


def test_calls_on_two_streams(dev):
    """Two calls at once, each on its own stream and workspace, give what they give alone."""
    gen, args = seeded(13), []
    for seed, lens in ((1, [(1, 3000)] * 4), (2, [(64, 900), (1, 2000)])):
        starts, lengths, table, pages = U.batch(lens, 64, seed)
        kp, vp, scales = to(dev, *C.random_cache(gen, pages, 2, 64, 256, BF16))
        q = rand(gen, int(starts[-1]), 16, 256).to(dev)
        args.append(((q, kp, vp, *to(dev, starts, lengths, table)), scales))
    alone = [A.paged_attention(*a, scales=s) for a, s in args]
    streams = [torch.cuda.Stream() for _ in args]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for stream, (a, s), g in zip(streams, args, got):
            with torch.cuda.stream(stream):
                g.append(A.paged_attention(*a, scales=s))
    torch.cuda.synchronize()
    for g, want in zip(got, alone):
        assert all(torch.equal(x, want) for x in g)


@pytest.mark.parametrize('lens,max_new', [([(1, 900), (2, 40), (1, 0)], 2), ([(130, 700)], 130),
                                          ([(40, 40), (1, 3000), (300, 300)], 300)])
def test_attention_in_place(dev, lens, max_new):
    """The output may be the queries or the gate themselves."""
    gen = seeded(21)
    starts, lengths, table, pages = U.batch(lens, 64)
    q, g = (rand(gen, int(starts[-1]), 16, 256).to(dev) for _ in range(2))
    kp, vp, scales = to(dev, *C.random_cache(gen, pages, 2, 64, 256, BF16))
    batch = to(dev, starts, lengths, table)
    want = A.paged_attention(q, kp, vp, *batch, gate=g, max_new=max_new, scales=scales)
    for pick in (0, 1):
        a = [q.clone(), g.clone()]
        got = A.paged_attention(a[0], kp, vp, *batch, gate=a[1], max_new=max_new, out=a[pick],
                                scales=scales)
        assert got is a[pick] and torch.equal(got, want)
