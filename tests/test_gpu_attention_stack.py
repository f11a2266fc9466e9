"""GPU tests of the attention blocks in MoEStack: the block against its formula in 64 bits
on its own intermediates, and the stack's chunked prefill and decode with attention layers."""
import pytest
import torch

from localmoe35ba3b_amd import router
from localmoe35ba3b_amd.convert import quantize_g128
from localmoe35ba3b_amd.operators import int8
from localmoe35ba3b_amd.runtime.attention import AttentionBlock, Batch
from localmoe35ba3b_amd.runtime.stack import SyntheticMoEStack
from tests import attention_util as U
from tests.conftest import BF16_TOL, assert_close, seeded

pytestmark = pytest.mark.gpu

H = 2048


def block(dev, seed, q_heads=16, kv_heads=2, dim=256, gated=True, pairs=32):
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)

    def bank(n, k):
        q, s = quantize_g128(torch.randn(n, k, generator=gen, device=dev) * 0.02)
        return {'q': q, 'scale': s}

    def weight(n):
        return torch.randn(n, generator=gen, device=dev) * 0.1

    rows = q_heads * dim * (2 if gated else 1) + 2 * kv_heads * dim
    return AttentionBlock(bank(rows, H), bank(H, q_heads * dim), q_heads, kv_heads, dim,
                          norm=weight(H), q_norm=weight(dim), k_norm=weight(dim),
                          inv_freq=U.frequencies(pairs).to(dev), gated=gated)


def ints(dev, *v):
    return torch.tensor(v, dtype=torch.int32, device=dev)


@pytest.mark.parametrize('gated,q_heads,kv_heads,dim', [(True, 16, 2, 256), (False, 12, 4, 128)])
def test_block_against_its_formula(dev, gated, q_heads, kv_heads, dim):
    """Two sequences, one with a history, and two padded rows: what the block adds is the
    output projection of 64-bit attention over its cache; padded rows stay as they are."""
    b = block(dev, 3, q_heads, kv_heads, dim, gated).allocate(9, 16)
    table = ints(dev, [4, 0, 7], [2, 8, 1])
    gen = seeded(4)
    past = torch.randn(20, H, generator=gen).to(torch.bfloat16).to(dev)
    b.forward_(past, Batch(ints(dev, 0, 0, 20), ints(dev, 0, 20), table))
    h = torch.randn(32, H, generator=gen).to(torch.bfloat16).to(dev)
    new = h.clone()
    batch = Batch(ints(dev, 0, 7, 30), ints(dev, 7, 43), table, 23)
    assert b.forward_(new, batch) is new
    assert torch.equal(new[30:], h[30:])
    # the projections as the block computes them, everything behind them in 64 bits
    x = int8.linear(router.rmsnorm(h, b.norm, b.eps), b.qkv['q'], b.qkv['scale']).cpu()
    q = x[:, :b.q_width].view(32, q_heads, -1)
    gate = q[..., dim:] if gated else None
    position = torch.cat([torch.arange(7), torch.arange(20, 43), torch.zeros(2)])
    q, _ = U.norm_rope(q[..., :dim], b.q_norm.cpu(), position, b.inv_freq.cpu())
    want, slack = U.attention(q.to(torch.bfloat16), b.k_pages.cpu(), b.v_pages.cpu(), *(
        t.cpu() for t in batch[:3]), gate=gate)
    w = b.o['q'].cpu().double() * b.o['scale'].cpu().double().repeat_interleave(128, 1)
    want, slack = want[:30].reshape(30, -1), slack[:30].reshape(30, -1)
    added, base = want @ w.t(), h[:30].double().cpu()
    # half a step of bf16 (2^-8) each for the residual sum and the projection's result, and for
    # every product one for the attention row and one for the dequantized weight
    step = 2.0 ** -8
    tol = step * ((base + added).abs() + added.abs()) + (slack + 2 * step * want.abs()) @ w.abs().t()
    assert ((new[:30].double().cpu() - base - added).abs() <= tol).all()
    # and the block's part of it is there: as much as 64-bit arithmetic adds, within 2 %
    assert_close((new[:30].double().cpu() - base).norm().numpy(), added.norm().numpy(), BF16_TOL)
    k, slack = U.norm_rope(x[:30, b.q_width:b.q_width + b.kv_width].view(30, kv_heads, dim),
                           b.k_norm.cpu(), position[:30], b.inv_freq.cpu())
    kept = U.gather(b.k_pages.cpu(), table[1].cpu(), 43, 16, 1)[20:]
    U.assert_rows(kept, k[7:30, 1], slack[7:30, 1], torch.bfloat16, 'keys of the cache')


@pytest.fixture(scope='module')
def stack(dev):
    st = SyntheticMoEStack(layers=3, seed=41, device=dev, max_tokens=64)
    st.attention = {l: block(dev, 50 + l).allocate(8, 16) for l in (0, 2)}
    return st


def prompt(dev, tokens, seed):
    return torch.randn(tokens, H, generator=seeded(seed)).to(torch.bfloat16).to(dev)


def run_layers(st, h, batch):
    for l in range(st.L):
        if l in st.attention:
            st.attention[l].forward_(h, batch)
        st.layer_forward(h, l)
    return h


def test_stack_runs_its_attention(dev, stack):
    """forward with attention is its blocks and layers one after another, bit for bit, for a
    prompt and for single tokens of a sequence that goes on."""
    table = ints(dev, [3, 1, 6])
    x = prompt(dev, 40, 1)
    one = Batch(ints(dev, 0, 40), ints(dev, 40), table, 40)
    assert torch.equal(stack.forward(x.clone(), batch=one), run_layers(stack, x.clone(), one))
    for step in range(3):
        y = prompt(dev, 1, 10 + step)
        one = Batch(ints(dev, 0, 1), ints(dev, 41 + step), table, 1)
        assert torch.equal(stack.forward(y.clone(), batch=one), run_layers(stack, y.clone(), one))


@pytest.mark.parametrize('tokens,chunk', [(100, 64), (70, 32)])
def test_stack_chunked_prefill(dev, stack, tokens, chunk):
    """Overlapped chunks give what the chunks give one after another, bit for bit, with the
    same cache behind them."""
    batch = Batch(ints(dev, 0, tokens), ints(dev, tokens), ints(dev, [5, 0, 2, 7, 1, 4, 6]))
    x = prompt(dev, tokens, tokens)
    want = stack.prefill(x, chunk, overlap=False, batch=batch)
    pages = [t.clone() for b in stack.attention.values() for t in (b.k_pages, b.v_pages)]
    used = [5, 0, 2, 7, 1, 4, 6][:-(-tokens // 16)]
    for b in stack.attention.values():
        b.k_pages.zero_(), b.v_pages.zero_()
    got = stack.prefill(x, chunk, batch=batch)
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    after = [t for b in stack.attention.values() for t in (b.k_pages, b.v_pages)]
    for a, b in zip(after, pages):
        a, b = (t[used].transpose(1, 2).reshape(-1, 2, 256)[:tokens] for t in (a, b))
        assert torch.equal(a, b)
    # and the second chunk saw the first: alone, it gives something else
    alone = Batch(ints(dev, 0, tokens - chunk), ints(dev, tokens - chunk), ints(dev, [3, 1, 0, 2, 4]))
    if tokens - chunk <= 64:
        assert not torch.equal(stack.forward(x[chunk:].clone(), batch=alone), want[chunk:])


def test_stack_decode_graph(dev, stack):
    """A captured decode step of three sequences follows their lengths between replays."""
    table = ints(dev, [0, 1], [2, 3], [4, 5])
    lengths = ints(dev, 3, 17, 9)
    batch = Batch(ints(dev, 0, 1, 2, 3), lengths, table, 1)
    for b in stack.attention.values():
        b.k_pages.normal_(), b.v_pages.normal_()
    h = prompt(dev, 3, 5)
    static = h.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        stack.forward(static, batch=batch)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        stack.forward(static, batch=batch)
    for step in range(4):
        x = prompt(dev, 3, 20 + step)
        lengths += 1
        static.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(static, run_layers(stack, x.clone(), batch))


def test_stack_refusals(dev, stack):
    x = prompt(dev, 4, 1)
    with pytest.raises(ValueError, match='batch'):
        stack.forward(x)
    with pytest.raises(ValueError, match='batch'):
        stack.prefill(x)
    two = Batch(ints(dev, 0, 2, 4), ints(dev, 2, 2), ints(dev, [0], [1]))
    with pytest.raises(ValueError, match='one sequence'):
        stack.prefill(x, batch=two)
    assert torch.equal(stack.forward(x.clone(), layers=0), x)
    with pytest.raises(RuntimeError, match='allocate'):
        block(dev, 1).forward_(x, two)
    with pytest.raises(ValueError, match='heads'):
        AttentionBlock(stack.attention[0].qkv, stack.attention[0].o, 8, 2, 256)


@pytest.mark.parametrize('tokens,chunk,first,end', [(100, 64, 0, 90), (100, 32, 5, 60), (90, 64, 70, 71)])
def test_stack_chunked_prefill_of_padded_rows(dev, stack, tokens, chunk, first, end):
    """Rows before and behind the sequence, whole chunks of them too, are none of its positions:
    bit for bit the chunks with batches written out by hand."""
    n = end - first
    table = ints(dev, [5, 0, 2, 7, 1, 4, 6])
    x = prompt(dev, tokens, tokens)
    past = prompt(dev, 3, 7)  # positions 0 .. 2
    stack.forward(past, batch=Batch(ints(dev, 0, 3), ints(dev, 3), table, 3))
    want = x.clone()
    for c0 in range(0, tokens, chunk):
        rows = min(chunk, tokens - c0)
        lo, hi = (min(max(v - c0, 0), rows) for v in (first, end))
        done = 3 + max(min(end, c0 + rows) - first, 0)
        stack.forward(want[c0:c0 + rows], batch=Batch(ints(dev, lo, hi), ints(dev, done), table, rows))
    batch = Batch(ints(dev, first, end), ints(dev, 3 + n), table)
    for overlap in (False, True):
        for b in stack.attention.values():
            b.k_pages.index_fill_(0, table[0, 1:].long(), 0)
        got = stack.prefill(x, chunk, overlap=overlap, batch=batch)
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_stack_without_rows(dev, stack):
    """A step of no token passes through the attention blocks."""
    batch = Batch(ints(dev, 0, 0), ints(dev, 5), ints(dev, [0]), 1)
    assert stack.attention[0].forward_(prompt(dev, 0, 1), batch).shape == (0, H)


def test_stack_refuses_before_it_writes(dev, stack):
    """Calls that one of the layers would refuse leave the rows and every cache as they were."""
    table, x = ints(dev, [5, 0, 2, 7, 1, 4, 6]), prompt(dev, 70, 9)
    caches = [t for b in stack.attention.values() for t in (b.k_pages, b.v_pages)]
    for t in caches:
        t.normal_()
    before, h = [t.clone() for t in caches], x.clone()
    good = Batch(ints(dev, 0, 70), ints(dev, 70), table)
    late, stack.attention[1] = block(dev, 1), block(dev, 1)  # without pages
    try:
        for run in (lambda b: stack.forward(h[:60], batch=b), lambda b: stack.prefill_(h, 32, batch=b),
                    lambda b: stack.prefill_(h, 32, overlap=False, batch=b)):
            with pytest.raises(RuntimeError, match='allocate'):
                run(good)
            stack.attention[1] = late.allocate(8, 16)
            with pytest.raises(ValueError, match='int32'):
                run(good._replace(lengths=good.lengths.long()))
            stack.attention[1] = block(dev, 1)
    finally:
        del stack.attention[1]
    with pytest.raises(MemoryError, match='token count'):
        stack.forward(h, batch=good)
    torch.cuda.synchronize()
    assert torch.equal(h, x) and all(torch.equal(a, b) for a, b in zip(caches, before))
    assert stack.prefill_(h, 32, batch=good) is h and not torch.equal(h, x)


@pytest.mark.parametrize('tokens,chunk', [(60, 32), (90, 32)])
def test_stack_prefill_graph(dev, stack, tokens, chunk):
    """A captured prefill of overlapped chunks, replayed with other rows and another length, with
    eager work in between."""
    table = ints(dev, [5, 0, 2, 7, 1, 4, 6])
    ends, lengths = ints(dev, 0, tokens), ints(dev, tokens)
    batch = Batch(ends, lengths, table)
    static = prompt(dev, tokens, 1)
    stack.prefill_(static, chunk, batch=batch)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        stack.prefill_(static, chunk, batch=batch)
    for step in range(4):
        x = prompt(dev, tokens, 30 + step)
        ends[1] = lengths[0] = tokens - 7 * step  # the rows behind are none of the sequence
        static.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        after = [t.clone() for b in stack.attention.values() for t in (b.k_pages, b.v_pages)]
        assert torch.equal(static, stack.prefill(x, chunk, overlap=False, batch=batch))
        torch.cuda.synchronize()
        eager = [t for b in stack.attention.values() for t in (b.k_pages, b.v_pages)]
        # as bits: pages that nothing wrote hold whatever was there, NaN among it
        assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(after, eager))
