"""GPU tests of the attention operators against 64-bit results: norms with rotation,
the paged append, paged attention, and the three run together as a program runs them."""
import math

import pytest
import torch

from localmoe35ba3b_amd.operators import attention as A
from tests import attention_util as U
from tests.conftest import seeded

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16
TYPES = pytest.mark.parametrize('dtype', [BF16, FP16])


def rand(gen, *shape, dtype=BF16, scale=1.0):
    return (torch.randn(shape, generator=gen) * scale).to(dtype)


def to(dev, *tensors):
    return [None if t is None else t.to(dev) for t in tensors]


# ------------------------------------------------------------------ norms and rotation
@TYPES
@pytest.mark.parametrize('tokens,q_heads,k_heads,dim,pairs', [
    (1, 16, 2, 256, 32), (5, 3, 1, 256, 128), (37, 32, 8, 128, 64), (6, 1, 1, 64, 8),
    (130, 7, 5, 64, 24), (4, 2, 2, 128, 0)])
def test_norm_rope(dev, tokens, q_heads, k_heads, dim, pairs, dtype):
    gen = seeded(tokens + dim)
    # a query and a gate of each head side by side; rows from tiny to large
    q = rand(gen, tokens, q_heads, 2 * dim, dtype=dtype)[..., :dim]
    k = rand(gen, tokens, k_heads, dim, dtype=dtype, scale=30.0)
    q[0, 0] = 0
    k[-1, -1] *= 1e-3
    qw, kw = torch.randn(dim, generator=gen) * 0.2, torch.randn(dim, generator=gen) * 0.2
    positions = torch.randint(0, 1 << 20, (tokens,), generator=gen)
    freq = U.frequencies(pairs) if pairs else None
    qd = torch.zeros(tokens, q_heads, 2 * dim, dtype=dtype, device=dev)
    qd[..., :dim] = q
    got = A.qk_norm_rope(qd[..., :dim], *to(dev, k, qw, kw, positions, freq))
    for g, x, w, what in zip(got, (q, k), (qw, kw), 'qk'):
        assert g.is_contiguous() and g.dtype == dtype
        U.assert_rows(g, *U.norm_rope(x, w, positions, freq), dtype, what)


def test_norm_rope_without_norm_and_layouts(dev):
    """No weights (no norm), negative and far positions, rows in another order, broadcast
    heads, rows off 16 bytes, and no tokens at all."""
    gen = seeded(3)
    q, k = rand(gen, 4, 33, 128), rand(gen, 33, 1, 128)
    positions = torch.arange(33) * 40_000 - 600_000
    freq = U.frequencies(16)
    qd, kd, pd, fd = to(dev, q, k, positions, freq)
    shifted = torch.empty(qd.numel() + 1, dtype=BF16, device=dev)[1:].view(33, 4, 128)
    shifted.copy_(qd.transpose(0, 1))
    a, b = A.qk_norm_rope(qd.transpose(0, 1), kd.expand(33, 6, 128), None, None, pd, fd)
    c, d = A.qk_norm_rope(shifted, kd, None, None, pd, fd)
    want = U.norm_rope(q.transpose(0, 1), None, positions, freq)
    U.assert_rows(a, *want, BF16, 'transposed')
    assert torch.equal(a, c) and torch.equal(b[:, 5:], d) and torch.equal(b[:, :1], d)
    q0, k0 = A.qk_norm_rope(qd[:, :0].transpose(0, 1), kd[:0], None, None, pd[:0], fd)
    assert q0.shape == (0, 4, 128) and k0.shape == (0, 1, 128)


def test_norm_rope_infinities_stay_in_their_row(dev):
    q = rand(seeded(4), 3, 2, 64)
    q[1, 0, 5] = math.inf
    q[2, 1, 7] = math.nan
    args = to(dev, q, rand(seeded(5), 3, 1, 64), torch.zeros(64), torch.zeros(64), torch.arange(3),
              U.frequencies(16))
    got, _ = A.qk_norm_rope(*args)
    assert got[1, 0].isnan().any() and got[2, 1].isnan().all()
    rest = torch.tensor([[1, 1], [0, 1], [1, 0]], dtype=torch.bool)
    want, slack = U.norm_rope(q, torch.zeros(64), torch.arange(3), U.frequencies(16))
    U.assert_rows(got.cpu()[rest], want[rest], slack[rest], BF16, 'other rows')


# ------------------------------------------------------------------ append
@TYPES
@pytest.mark.parametrize('lens,page,q_heads,heads,dim,pairs', [
    ([(1, 1)], 16, 16, 2, 256, 32),
    ([(1, 17), (1, 16), (0, 9), (1, 100)], 16, 4, 2, 128, 64),
    ([(40, 40), (3, 130), (1, 64), (0, 0), (70, 71)], 64, 6, 3, 64, 16),
    ([(33, 1000)], 1024, 0, 1, 256, 0)])
def test_append(dev, lens, page, q_heads, heads, dim, pairs, dtype):
    gen = seeded(page + dim)
    starts, lengths, table, pages = U.batch(lens, page)
    tokens, live = int(starts[-1]) + 3, int(starts[-1])  # three rows of no sequence
    k, v = rand(gen, tokens, heads, dim, dtype=dtype), rand(gen, tokens, heads, dim, dtype=dtype)
    q = rand(gen, tokens, q_heads, dim, dtype=dtype) if q_heads else None
    kw, qw = torch.randn(dim, generator=gen) * 0.1, torch.randn(dim, generator=gen) * 0.1
    freq = U.frequencies(pairs) if pairs else None
    kp, vp = (rand(gen, pages, heads, page, dim, dtype=dtype) for _ in range(2))
    kd, vd = to(dev, kp, vp)
    got = A.append(kd, vd, *to(dev, k, v, starts, lengths, table), inv_freq=to(dev, freq)[0],
                   k_weight=kw.to(dev), q=to(dev, q)[0], q_weight=qw.to(dev))
    positions = torch.cat([torch.arange(n - c, n) for c, n in lens])
    want, slack = U.norm_rope(k[:live], kw, positions, freq)
    wrote = torch.zeros(kp.shape, dtype=torch.bool)
    kc, vc, row = kd.cpu(), vd.cpu(), 0
    for s, (count, n) in enumerate(lens):
        for p in range(n - count, n):
            at = (int(table[s, p // page]), slice(None), p % page)
            U.assert_rows(kc[at], want[row], slack[row], dtype, f'key {s} {p}')
            assert torch.equal(vc[at], v[row])
            wrote[at] = True
            row += 1
    assert torch.equal(kc[~wrote], kp[~wrote]) and torch.equal(vc[~wrote], vp[~wrote])
    if q is None:
        assert got is None
    else:
        U.assert_rows(got[:live], *U.norm_rope(q[:live], qw, positions, freq), dtype, 'queries')
        assert not got[live:].any()


def test_append_outside_the_table_is_not_written(dev):
    """Positions before 0 or behind the table's pages, and page numbers out of range."""
    k, v = rand(seeded(1), 8, 1, 64), rand(seeded(2), 8, 1, 64)
    pages = torch.zeros(3, 1, 16, 64, dtype=BF16, device=dev)
    starts = torch.tensor([0, 4, 8], dtype=torch.int32)
    lengths = torch.tensor([2, 34], dtype=torch.int32)  # positions -2 .. 1 and 30 .. 33
    table = torch.tensor([[0, 1], [2, 99]], dtype=torch.int32)  # 99 is taken as the last page
    kp, vp = pages.clone(), pages.clone()
    A.append(kp, vp, *to(dev, k, v, starts, lengths, table))
    want = pages.cpu()
    want[0, 0, :2] = v[2:4, 0]
    want[2, 0, 14:] = v[4:6, 0]
    assert torch.equal(vp.cpu(), want)


# ------------------------------------------------------------------ attention
def attend(dev, lens, page, q_heads, heads, dim, dtype, gate=False, pad=0, seed=0, scale=None,
           max_new=None, sharp=1.0):
    gen = seeded(seed)
    starts, lengths, table, pages = U.batch(lens, page, seed)
    tokens = int(starts[-1]) + pad
    q = rand(gen, tokens, q_heads, dim, dtype=dtype, scale=sharp)
    g = rand(gen, tokens, q_heads, dim, dtype=dtype) if gate else None
    kp, vp = (rand(gen, pages, heads, page, dim, dtype=dtype) for _ in range(2))
    # what no sequence holds must not matter, whatever it is
    held = torch.zeros(pages, page, dtype=torch.bool)
    for s, (_, n) in enumerate(lens):
        for p in range(n):
            held[int(table[s, p // page]), p % page] = True
    kd, vd = kp.transpose(1, 2).clone(), vp.transpose(1, 2).clone()
    kd[~held], vd[~held] = math.nan, math.inf
    kd, vd = (x.transpose(1, 2).contiguous().to(dev) for x in (kd, vd))
    before = torch.full(q.shape, 7.0, dtype=dtype, device=dev)
    out = before.clone()
    args = to(dev, q, kd, vd, starts, lengths, table)
    got = A.paged_attention(*args, scale=scale, gate=to(dev, g)[0], max_new=max_new, out=out)
    assert got is out
    U.assert_attention(got, U.attention(q, kp, vp, starts, lengths, table, scale, g),
                       f'{lens} {page} {q_heads}/{heads} {dim}', before)
    return args, to(dev, g)[0], got


DECODE = [
    ([(1, 1)], 16, 16, 2, 256), ([(1, 2), (1, 17), (1, 63), (1, 64), (1, 65)], 16, 8, 2, 128),
    ([(1, 1000)], 64, 8, 1, 256), ([(1, 700), (1, 1), (0, 5), (1, 0), (1, 333)], 32, 4, 4, 64),
    ([(2, 500), (1, 90), (2, 2)], 16, 16, 2, 256), ([(16, 300), (3, 40)], 64, 1, 1, 64),
    ([(1, 600)] * 20, 128, 3, 1, 128), ([(1, 520), (1, 31)], 32, 20, 1, 64)]
CHUNKS = [
    ([(33, 33)], 16, 16, 2, 256), ([(70, 200)], 64, 4, 2, 128), ([(17, 17), (50, 350)], 32, 3, 3, 64),
    ([(130, 131), (1, 400), (0, 0), (9, 9), (2, 77)], 16, 8, 1, 256),
    ([(20, 500)], 1024, 32, 8, 128), ([(5, 3), (40, 39)], 16, 6, 2, 64), ([(9, 300)], 64, 40, 1, 128)]


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
    """Weights from equal to a single one, where the running maximum grows by large steps."""
    attend(dev, [(1, 700), (60, 400)], 16, 8, 2, 128, dtype, sharp=sharp, scale=0.11)


def test_attention_negative_and_zero_scale(dev):
    for scale in (0.0, -0.2):
        attend(dev, [(1, 90), (20, 130)], 16, 4, 2, 64, BF16, scale=scale)


def test_attention_growing_scores(dev):
    """Every key scores above all before it: the running maximum moves at every step."""
    n, dim = 512, 64
    k = torch.zeros(n // 16, 1, 16, dim)
    k[..., 0] = torch.arange(n).view(-1, 1, 16) / 4
    v = rand(seeded(8), n // 16, 1, 16, dim)
    q = torch.zeros(40, 1, dim)
    q[..., 0] = 1.0
    k, q = k.to(BF16), q.to(BF16)
    table = torch.arange(n // 16, dtype=torch.int32)[None].expand(2, -1)
    starts = torch.tensor([0, 1, 40], dtype=torch.int32)
    lengths = torch.tensor([n, n], dtype=torch.int32)
    got = A.paged_attention(*to(dev, q, k, v, starts, lengths, table), scale=1.0)
    U.assert_attention(got, U.attention(q, k, v, starts, lengths, table, 1.0), 'growing')


@pytest.mark.parametrize('new', [1, 40])
def test_attention_later_values_do_not_reach_earlier_rows(dev, new):
    """Infinities and NaN among the keys and values of a position show in the rows that see
    it and in no other."""
    lens = [(new, 100), (new, 70)]
    gen = seeded(6)
    starts, lengths, table, pages = U.batch(lens, 16)
    q = rand(gen, 2 * new, 4, 64)
    kp, vp = (rand(gen, pages, 2, 16, 64) for _ in range(2))
    clean = U.attention(q, kp, vp, starts, lengths, table)
    bad = 100 - max(1, new // 2)  # a position of sequence 0 that its last rows see
    at = int(table[0, bad // 16])
    vp[at, 0, bad % 16, 3], vp[at, 0, bad % 16, 40] = math.inf, math.nan
    kp[at, 1, bad % 16, 9] = math.nan
    got = A.paged_attention(*to(dev, q, kp, vp, starts, lengths, table)).cpu()
    sees = torch.zeros(2 * new, 4, 64, dtype=torch.bool)
    rows = slice(max(0, new - (100 - bad)), new)
    sees[rows, :2, 3] = sees[rows, :2, 40] = True
    sees[rows, 2:] = True
    assert not got[sees].isfinite().any()
    U.assert_rows(got[~sees], clean[0][~sees], clean[1][~sees], BF16, 'rows before it')


def test_attention_malformed_batches_stay_in_bounds(dev):
    """Page numbers, lengths and starts out of range: some result, no access outside."""
    q, kp, vp = to(dev, rand(seeded(1), 40, 4, 64), rand(seeded(2), 5, 2, 16, 64),
                   rand(seeded(3), 5, 2, 16, 64))
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)
    table = ints([0, 99, -3], [1, 2, 2 ** 31 - 1])
    for starts, lengths in ((ints(0, 20, 40), ints(1000, -5)), (ints(0, 30, 100), ints(48, 48)),
                            (ints(-9, 20, 10), ints(48, 40)), (ints(50, 60, 70), ints(4, 4)),
                            (ints(0, 1, 2), ints(2 ** 31 - 1, -2 ** 31))):
        for max_new in (1, 40):
            A.paged_attention(q, kp, vp, starts, lengths, table, max_new=max_new)
            torch.cuda.synchronize()


def test_attention_layouts(dev):
    """Strided queries and gates, pages of one tensor that holds both, a shared page table."""
    gen = seeded(9)
    lens, heads, dim, page = [(1, 90), (1, 90), (1, 90)], 2, 128, 16
    both = rand(gen, 7, 2, heads, page, dim)
    row = torch.randperm(7, generator=gen)[:6].to(torch.int32)
    starts = torch.arange(4, dtype=torch.int32)
    lengths = torch.tensor([90, 50, 1], dtype=torch.int32)
    qg = rand(gen, 8, 3, 2 * dim).transpose(0, 1)  # heads before tokens
    bd, rd, sd, ld, qd = to(dev, both, row, starts, lengths, qg)
    got = A.paged_attention(qd[..., :dim], bd[:, 0], bd[:, 1], sd, ld, rd.expand(3, 6),
                            gate=qd[..., dim:], max_new=1)
    U.assert_attention(got, U.attention(qg[..., :dim], both[:, 0], both[:, 1], starts, lengths,
                                        row.expand(3, 6), gate=qg[..., dim:]), 'strided')


def test_attention_far_pages(dev):
    """Offsets beyond 32 bits: 4.3 GB of keys, of which a sequence's pages lie at the end."""
    heads, page, dim, n = 2, 1024, 256, 1500
    pages = (1 << 32) // (heads * page * dim * 2) + 3
    kd = torch.empty(pages, heads, page, dim, dtype=BF16, device=dev)
    vd = torch.empty(pages, heads, page, dim, dtype=BF16, device=dev)
    gen = seeded(10)
    k, v = rand(gen, 2, heads, page, dim), rand(gen, 2, heads, page, dim)
    kd[-2:], vd[-2:] = to(dev, k, v)
    starts, lengths = torch.tensor([0, 1, 30], dtype=torch.int32), torch.tensor([n, n], dtype=torch.int32)
    q = rand(gen, 30, 4, dim)
    table = torch.tensor([[0, 1], [1, 0]], dtype=torch.int32)
    got = A.paged_attention(*to(dev, q), kd, vd, *to(dev, starts, lengths, table + pages - 2))
    U.assert_attention(got, U.attention(q, k, v, starts, lengths, table), 'far pages')
    new_k, new_v = rand(gen, 2, heads, dim), rand(gen, 2, heads, dim)
    A.append(kd, vd, *to(dev, new_k, new_v, torch.tensor([0, 1, 2], dtype=torch.int32), lengths,
                         table + pages - 2))
    assert torch.equal(vd[-1, :, (n - 1) % page].cpu(), new_v[0])
    assert torch.equal(vd[-2, :, (n - 1) % page].cpu(), new_v[1])


# ------------------------------------------------------------------ the three together
def step(cache, q, k, v, gate, qw, kw, freq, batch, max_new):
    q = A.append(*cache, k, v, *batch, inv_freq=freq, k_weight=kw, q=q, q_weight=qw)
    return A.paged_attention(q, *cache, *batch, gate=gate, max_new=max_new)


@TYPES
def test_prompt_in_chunks_then_tokens(dev, dtype):
    """A prompt appended in ragged chunks, then tokens one at a time, against attention over
    the whole sequence at once: the cache holds what the keys and values of each call were."""
    gen, dim, hq, hk, page, total = seeded(11), 128, 6, 2, 16, 90
    q, k, v, gate = (rand(gen, total, h, dim, dtype=dtype) for h in (hq, hk, hk, hq))
    qw, kw, freq = torch.randn(dim, generator=gen) * 0.1, torch.randn(dim, generator=gen) * 0.1, \
        U.frequencies(32)
    cache = [torch.full((8, hk, page, dim), math.nan, dtype=dtype, device=dev) for _ in range(2)]
    table = torch.tensor([[5, 0, 7, 1, 3, 2]], dtype=torch.int32, device=dev)
    parts, at = [], 0
    weights = to(dev, qw, kw, freq)
    for count in (37, 1, 2, 46, 1, 1, 1, 1):
        rows = slice(at, at + count)
        at += count
        batch = (torch.tensor([0, count], dtype=torch.int32, device=dev),
                 torch.tensor([at], dtype=torch.int32, device=dev), table)
        parts.append(step(cache, *to(dev, q[rows], k[rows], v[rows], gate[rows]), *weights, batch,
                          count))
    positions = torch.arange(total)
    qn, q_slack = U.norm_rope(q, qw, positions, freq)
    kn, k_slack = U.norm_rope(k, kw, positions, freq)
    # the cache's keys are what attention sees: compare on them, after checking them
    kc = cache[0].cpu()[table[0].cpu().long()].transpose(1, 2).reshape(-1, hk, dim)[:total]
    U.assert_rows(kc, kn, k_slack, dtype, 'keys')
    qs, _ = A.qk_norm_rope(*to(dev, q, k, qw, kw, positions, freq))
    U.assert_rows(qs, qn, q_slack, dtype, 'queries')
    one = torch.tensor([0, total], dtype=torch.int32), torch.tensor([total], dtype=torch.int32)
    want = U.attention(qs.cpu(), cache[0].cpu(), cache[1].cpu(), *one, table.cpu(), gate=gate)
    U.assert_attention(torch.cat(parts), want, 'chunks and tokens')


def test_captured_step_follows_its_batch(dev):
    """A captured decode step replayed while lengths and inputs change between replays, with
    eager work of the same operators in between; two graphs alive at once."""
    gen, dim, hq, hk, page = seeded(12), 256, 16, 2, 16
    cache = [rand(gen, 40, hk, page, dim).to(dev) for _ in range(2)]
    starts = torch.arange(4, dtype=torch.int32, device=dev)
    lengths = torch.tensor([5, 170, 33], dtype=torch.int32, device=dev)
    table = torch.randperm(40, generator=gen)[:36].view(3, 12).to(dev, torch.int32)
    ins = [rand(gen, 3, h, dim).to(dev) for h in (hq, hk, hk, hq)]
    weights = to(dev, torch.zeros(dim), torch.zeros(dim), U.frequencies(32))
    batch = (starts, lengths, table)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(cache, *ins, *weights, batch, 1)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(cache, *ins, *weights, batch, 1)
        graphs.append((graph, out))
    for i in range(6):
        lengths += 1
        for x in ins:
            x.copy_(rand(gen, *x.shape))
        graph, out = graphs[i % 2]
        graph.replay()
        eager = [c.clone() for c in cache]
        want = step(eager, *ins, *weights, batch, 1)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert all(torch.equal(a, b) for a, b in zip(cache, eager))


def test_calls_on_two_streams(dev):
    """Two calls at once, each on its own stream and workspace, give what they give alone."""
    gen = seeded(13)
    args = []
    for seed, lens in ((1, [(1, 3000)] * 4), (2, [(64, 900), (1, 2000)])):
        starts, lengths, table, pages = U.batch(lens, 64, seed)
        q = rand(gen, int(starts[-1]), 16, 256)
        args.append(to(dev, q, *(rand(gen, pages, 2, 64, 256) for _ in range(2)), starts, lengths,
                       table))
    alone = [A.paged_attention(*a) for a in args]
    streams = [torch.cuda.Stream() for _ in args]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for s, a, g in zip(streams, args, got):
            with torch.cuda.stream(s):
                g.append(A.paged_attention(*a))
    torch.cuda.synchronize()
    for g, want in zip(got, alone):
        assert all(torch.equal(x, want) for x in g)


def test_append_without_sequences(dev):
    """Every row is one of no sequence: zeros for the queries, the cache as it was."""
    kp = rand(seeded(1), 4, 2, 16, 64).to(dev)
    q, k = rand(seeded(2), 5, 4, 64).to(dev), rand(seeded(3), 5, 2, 64).to(dev)
    none, before = torch.zeros(1, dtype=torch.int32, device=dev), kp.clone()
    torch.full((5, 4, 64), 3.0, dtype=BF16, device=dev)  # memory that is not 0
    got = A.append(kp, kp.clone(), k, k, none, none[:0], none[:0].view(0, 1), q=q)
    assert not got.any() and torch.equal(kp, before)
    assert not A.paged_attention(q, kp, kp, none, none[:0], none[:0].view(0, 1)).any()


@pytest.mark.parametrize('sequences', [70, 300, 600])
@pytest.mark.parametrize('chunks', [False, True])
def test_attention_many_sequences(dev, sequences, chunks):
    """More sequences than a wave or a workgroup looks at together; some without new tokens,
    some without a visible key, with chunks among them."""
    gen = torch.Generator().manual_seed(sequences)
    length = torch.randint(0, 90, (sequences,), generator=gen).tolist()
    lens = [(i % 4 if i % 7 else 30 * chunks, n) for i, n in enumerate(length)]
    lens = [(new, max(n, new - 1)) for new, n in lens]
    attend(dev, lens, 16, 4, 2, 64, BF16, gate=chunks, pad=2, seed=sequences,
           max_new=max(n for n, _ in lens))


def long_cache(dev, heads, keys, dim, seed):
    """A cache of one sequence in random pages, made on the GPU, and its CPU copy."""
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    pages = -(-keys // 64)
    kp, vp = (torch.randn(pages, heads, 64, dim, generator=gen, device=dev).to(BF16) for _ in range(2))
    table = torch.randperm(pages, generator=seeded(seed)).to(torch.int32)[None]
    return kp, vp, table


@pytest.mark.parametrize('new,heads,keys,dim', [(2, 128, 18000, 64), (2, 128, 27000, 64), (1, 128, 9000, 256),
                                                (20, 128, 10000, 64), (20, 128, 4700, 256)])
def test_attention_long_parts(dev, new, heads, keys, dim):
    """Parts of a sequence longer than the pages that a wave looks up at a time: as many heads
    as this leave each few parts."""
    kp, vp, table = long_cache(dev, heads, keys, dim, keys)
    q = rand(seeded(keys), new, heads, dim)
    batch = torch.tensor([0, new], dtype=torch.int32), torch.tensor([keys], dtype=torch.int32), table
    got = A.paged_attention(q.to(dev), kp, vp, *to(dev, *batch))
    some = [0, heads // 2, heads - 1]  # heads are independent: three of them in 64 bits
    want = U.attention(q[:, some], kp[:, some].cpu(), vp[:, some].cpu(), *batch)
    U.assert_attention(got[:, some], want, f'{new} {heads} {keys} {dim}')
    assert got.isfinite().all()


@TYPES
@pytest.mark.parametrize('dim', [128, 256])
@pytest.mark.parametrize('new', [1, 40])
def test_attention_odd_values_of_all_types(dev, new, dim, dtype):
    """Infinities and NaN among the values of a position that only the last rows see."""
    lens = [(new, 100), (new, 70)]
    gen = seeded(dim + new)
    starts, lengths, table, pages = U.batch(lens, 16)
    q = rand(gen, 2 * new, 4, dim, dtype=dtype)
    kp, vp = (rand(gen, pages, 2, 16, dim, dtype=dtype) for _ in range(2))
    clean = U.attention(q, kp, vp, starts, lengths, table)
    bad = 100 - max(1, new // 2)
    at = int(table[0, bad // 16])
    vp[at, 0, bad % 16, 3], vp[at, 0, bad % 16, dim - 2] = math.inf, math.nan
    vp[at, 1, bad % 16, 64] = -math.inf
    kp[at, 1, bad % 16, 9] = math.nan
    got = A.paged_attention(*to(dev, q, kp, vp, starts, lengths, table)).cpu()
    sees = torch.zeros(2 * new, 4, dim, dtype=torch.bool)
    rows = slice(max(0, new - (100 - bad)), new)
    sees[rows, :2, 3] = sees[rows, :2, dim - 2] = True
    sees[rows, 2:] = True
    assert not got[sees].isfinite().any()
    U.assert_rows(got[~sees], clean[0][~sees], clean[1][~sees], dtype, 'rows before it')


@pytest.mark.parametrize('lens,max_new', [([(1, 900), (2, 40), (1, 0)], 2), ([(130, 700)], 130),
                                          ([(40, 40), (1, 3000), (300, 300)], 300)])
def test_attention_in_place(dev, lens, max_new):
    """The output may be the queries or the gate themselves."""
    gen = seeded(21)
    starts, lengths, table, pages = U.batch(lens, 64)
    q, g = (rand(gen, int(starts[-1]), 16, 256).to(dev) for _ in range(2))
    cache = to(dev, *(rand(gen, pages, 2, 64, 256) for _ in range(2)), starts, lengths, table)
    want = A.paged_attention(q, *cache, gate=g, max_new=max_new)
    for pick in (0, 1):
        a = [q.clone(), g.clone()]
        got = A.paged_attention(a[0], *cache, gate=a[1], max_new=max_new, out=a[pick])
        assert got is a[pick] and torch.equal(got, want)


def test_attention_on_another_stream_than_its_tensors(dev):
    """A call on a stream that has waited for its inputs' stream; the output is made there."""
    gen = seeded(23)
    starts, lengths, table, pages = U.batch([(1, 500), (70, 300)], 16)
    args = to(dev, rand(gen, 71, 8, 128), *(rand(gen, pages, 2, 16, 128) for _ in range(2)), starts,
              lengths, table)
    want = A.paged_attention(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = A.paged_attention(*args)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_two_captured_calls_replayed_in_turn(dev):
    """Two graphs of one pool, one after another: each call's workspace is its own."""
    gen = seeded(25)
    graphs, outs, wants = [], [], []
    args = []
    for seed, lens in ((1, [(1, 2000)] * 3), (2, [(50, 400), (1, 900)])):
        starts, lengths, table, pages = U.batch(lens, 64, seed)
        args.append(to(dev, rand(gen, int(starts[-1]), 16, 256),
                       *(rand(gen, pages, 2, 64, 256) for _ in range(2)), starts, lengths, table))
    wants = [A.paged_attention(*a) for a in args]
    torch.cuda.synchronize()
    for a in args:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=graphs[0].pool() if graphs else None):
            outs.append(A.paged_attention(*a))
        graphs.append(graph)
    for _ in range(3):
        for graph, out, want, a in zip(graphs, outs, wants, args):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)
            A.paged_attention(*a)  # eager work between replays


@pytest.mark.parametrize('sequences,longest,dim', [(70, 900, 64), (70, 700, 256), (5, 5000, 128),
                                                   (270, 600, 64)])
def test_attention_unequal_tiles(dev, sequences, longest, dim):
    """Tiles whose keys differ by far, split into different counts of parts, some into none; more
    sequences than a wave or a workgroup looks at together."""
    gen = torch.Generator().manual_seed(longest)
    lens = []
    for i in range(sequences):
        n = longest if i % 17 == 3 else int(torch.randint(1, 120, (1,), generator=gen))
        lens.append((min(n, 10 + i % 13), n))
    attend(dev, lens, 16, 6, 2, dim, BF16, gate=True, pad=1, seed=longest)


@pytest.mark.parametrize('dim', [64, 128, 256])
@pytest.mark.parametrize('new,past,sink', [(1, 3000, 0), (1, 3000, 1500), (3, 2000, 5), (40, 2000, 0),
                                           (150, 4000, 700)])
def test_attention_fp16_tails_of_small_weights(dev, new, past, sink, dim):
    """One key far above the rest, whose own values are 0: the result is the others' weights, which
    are 2^-25 of the largest.  They stay apart from 0 although fp16 ends at 2^-24.

    attention()'s fp16 tolerance takes a weight as off by half of fp16's smallest step, 2^-25, in a
    sum of at least 1.  The kernels' weights are 2^7 times as large, so that half step is 2^-32 of
    the sum: that is what a value counts for here."""
    gen = seeded(dim + new)
    n = past + new
    starts, lengths, table, pages = U.batch([(new, n)], 64, dim)
    q, kp, vp = torch.zeros(new, 4, dim), torch.zeros(pages, 2, 64, dim), torch.zeros(pages, 2, 64, dim)
    q[..., 0] = 4.0
    vp[:] = 1.0 + 0.25 * torch.randn(vp.shape, generator=gen)
    at = int(table[0, sink // 64])
    kp[at, 0, sink % 64, 0], kp[at, 1, sink % 64, 0] = 17.25 / 4, 17.5 / 4  # 2^-24.9 and 2^-25.2
    vp[at, :, sink % 64] = 0
    q, kp, vp = q.to(FP16), kp.to(FP16), vp.to(FP16)
    for extra in (0, 1):  # alone, and beside a sequence of its own length
        if extra:
            starts = torch.tensor([0, new, new + 1], dtype=torch.int32)
            lengths, table = torch.tensor([n, n], dtype=torch.int32), table.expand(2, -1)
            q = torch.cat([q, q[-1:]])
        got = A.paged_attention(*to(dev, q, kp, vp, starts, lengths, table), scale=1.0)
        ref, slack = U.attention(q, kp, vp, starts, lengths, table, 1.0)
        sums = [U.gather(vp, table[0], n, 64, h).double().abs().cumsum(0) for h in range(2)]
        for t in range(new + extra):
            seen = past + min(t, new - 1)
            for h in range(4):
                slack[t, h] -= (2.0 ** -25 - 2.0 ** -32) * sums[h // 2][seen]
        assert (slack > 0).all()
        U.assert_attention(got, (ref, slack), f'{new} {past} {sink} {dim}')


@TYPES
@pytest.mark.parametrize('new', [1, 40])
def test_attention_gates_from_far_to_far(dev, new, dtype):
    """Values of every mantissa under gates to both ends of their range.  Scores of 0 leave the
    attention exact but for its exponential (2 steps of 2^-24), the division and a product (a step
    each); the gate adds (1.25 |x| + 5) steps and a product.  Rounding is monotone: a result lies
    between the roundings of that interval's ends."""
    gates = [-87.0, -80.0, -60.5, -45.0, -33.25, -17.0, -9.5, -3.0, -1.0, -0.125, 0.0, 0.3, 2.0, 7.0,
             20.0, 200.0, math.inf, -200.0, -math.inf]
    heads, dim = len(gates), 128
    g = torch.tensor(gates).to(dtype)[None, :, None].expand(new, heads, dim)
    v = (1 + torch.arange(dim) / dim).to(dtype)
    pages = torch.zeros(3, 1, 16, dim, dtype=dtype)
    starts, lengths = torch.tensor([0, new], dtype=torch.int32), torch.tensor([new], dtype=torch.int32)
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32)
    q = torch.randn(new, heads, dim, generator=seeded(new)).to(dtype)
    got = A.paged_attention(*to(dev, q, pages, v.expand_as(pages).contiguous(), starts, lengths, table),
                            gate=to(dev, g)[0]).cpu()
    x = g.double()
    want = v.double() * torch.sigmoid(x)
    slack = torch.where(x.isinf(), 0.0, (1.25 * x.abs() + 10) * 2.0 ** -24)
    low, high = (want * (1 - slack)).to(dtype), (want * (1 + slack)).to(dtype)
    assert ((got >= low) & (got <= high)).all()
    assert torch.equal(got[:, 16], v.expand(new, dim)) and not got[:, 17:].any()


def test_one_token_and_one_head_of_odd_pitch(dev):
    """One token of rows 260 apart, one head, and pages whose single head was transposed into place
    give what contiguous copies of them give."""
    gen = seeded(31)
    rows = rand(gen, 3, 2 * 128 + 4).to(dev)
    kv = rand(gen, 3, 128 + 4).to(dev)
    cache = [rand(gen, 9, 16, 1, 128).to(dev).transpose(1, 2) for _ in range(2)]
    plain = [c.clone(memory_format=torch.contiguous_format).view(-1).view(9, 1, 16, 128) for c in cache]
    lengths = torch.tensor([100], dtype=torch.int32)
    table = torch.tensor([[3, 1, 8, 0, 2, 7, 5]], dtype=torch.int32)
    for count in (1, 3):
        batch = to(dev, torch.tensor([0, count], dtype=torch.int32), lengths, table)
        q = rows[:count, :256].view(count, 2, 128)
        k = kv[:count, :128].view(count, 1, 128)
        odd = step(cache, q, k, k, q, None, None, None, batch, count)
        want = step(plain, *(t.clone(memory_format=torch.contiguous_format) for t in (q, k, k, q)),
                    None, None, None, batch, count)
        assert torch.equal(odd, want) and all(torch.equal(a, b) for a, b in zip(cache, plain))
        a, b = A.qk_norm_rope(q, k, None, None, torch.arange(count, device=dev), None)
        assert torch.equal(a, q) and torch.equal(b, k)
