"""GPU tests of the attention block with a cache in 8 bits, positions of several axes and W8A8
projections, alone and in the stack."""
import pytest
import torch

from localmoe35ba3b_amd.operators import attention as A
from localmoe35ba3b_amd.operators import int8, w8a8
from localmoe35ba3b_amd import router
from localmoe35ba3b_amd.runtime.attention import Batch
from localmoe35ba3b_amd.runtime.stack import SyntheticMoEStack
from tests import attention_util as U
from tests import cache8_util as C
from tests.conftest import BF16_TOL, assert_close, seeded
from tests.test_gpu_attention_stack import H, block, ints, prompt, run_layers

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn


def eight(dev, seed, w8a8=False, pages=8, **change):
    b = block(dev, seed, **change)
    b.axes = (torch.arange(32, device=dev) % 3).to(torch.int32)
    b.w8a8 = w8a8
    return b.allocate(pages, 16, E4M3)


def grid(dev, first, tokens):
    at = torch.arange(first, first + tokens, device=dev)
    return torch.stack([at // 24, at % 24 // 6, at % 6])


@pytest.mark.parametrize('wide', [False, True])
@pytest.mark.parametrize('gated,q_heads,kv_heads,dim', [(True, 16, 2, 256), (False, 12, 4, 128)])
def test_block_against_its_formula(dev, gated, q_heads, kv_heads, dim, wide):
    """Two sequences, one with a history, and two padded rows: what the block adds is the output
    projection of 64-bit attention over what its cache holds; padded rows stay as they are."""
    b = eight(dev, 3, wide, 9, q_heads=q_heads, kv_heads=kv_heads, dim=dim, gated=gated)
    table = ints(dev, [4, 0, 7], [2, 8, 1])
    gen = seeded(4)
    past = torch.randn(20, H, generator=gen).to(torch.bfloat16).to(dev)
    b.forward_(past, Batch(ints(dev, 0, 0, 20), ints(dev, 0, 20), table, None, grid(dev, 0, 20)))
    h = torch.randn(32, H, generator=gen).to(torch.bfloat16).to(dev)
    new = h.clone()
    positions = torch.cat([grid(dev, 0, 7), grid(dev, 20, 23), grid(dev, 0, 2)], 1)
    batch = Batch(ints(dev, 0, 7, 30), ints(dev, 7, 43), table, 23, positions)
    b.check(h, batch)
    assert b.forward_(new, batch) is new
    assert torch.equal(new[30:], h[30:])
    if wide:
        x = w8a8.gemm(*w8a8.norm_quantize(h, b.norm, b.eps), b.qkv['q'], b.qkv['scale'])
    else:
        x = int8.linear(router.rmsnorm(h, b.norm, b.eps), b.qkv['q'], b.qkv['scale'])
    q, k, _ = x.split([b.q_width, b.kv_width, b.kv_width], 1)
    q, gate = q.view(32, q_heads, -1), None
    if gated:
        q, gate = q[..., :dim], q[..., dim:].cpu()
    q, _ = A.qk_norm_rope(q, k.view(32, kv_heads, dim), b.q_norm, b.k_norm, positions, b.inv_freq,
                          b.eps, b.axes)
    want, slack = U.attention(q.cpu(), *C.held(b.k_pages, b.v_pages, b.scales, torch.bfloat16),
                              *(t.cpu() for t in batch[:3]), gate=gate)
    w = b.o['q'].cpu().double() * b.o['scale'].cpu().double().repeat_interleave(128, 1)
    want, slack = want[:30].reshape(30, -1), slack[:30].reshape(30, -1)
    added, base = want @ w.t(), h[:30].double().cpu()
    # half a step of bf16 (2^-8) each for the residual sum and the projection's result; for every
    # product one for the attention row and, in W8A16, one for the dequantized weight, in W8A8 half a
    # step of the row's quantization (1 / 254 of its group's largest value, 2^-7 of which it is off by)
    step = 2.0 ** -8
    off = slack + 2 * step * want.abs()
    if wide:
        top = (want.abs() * (1 + step) + slack).view(30, -1, 128).amax(-1, keepdim=True)
        off = off + (top / 254 * 1.01).expand(-1, -1, 128).reshape(30, -1)
    tol = step * ((base + added).abs() + added.abs()) + off @ w.abs().t()
    assert ((new[:30].double().cpu() - base - added).abs() <= tol).all()
    assert_close((new[:30].double().cpu() - base).norm().numpy(), added.norm().numpy(), BF16_TOL)


@pytest.fixture(scope='module')
def stack(dev):
    st = SyntheticMoEStack(layers=3, seed=41, device=dev, max_tokens=64)
    st.attention = {l: eight(dev, 50 + l, w8a8=l == 2) for l in (0, 2)}
    return st


def test_stack_runs_its_attention(dev, stack):
    """forward is its blocks and layers one after another, bit for bit, for a prompt and for single
    tokens of a sequence that goes on."""
    table = ints(dev, [3, 1, 6])
    x = prompt(dev, 40, 1)
    one = Batch(ints(dev, 0, 40), ints(dev, 40), table, 40, grid(dev, 0, 40))
    assert torch.equal(stack.forward(x.clone(), batch=one), run_layers(stack, x.clone(), one))
    for step in range(3):
        y = prompt(dev, 1, 10 + step)
        one = Batch(ints(dev, 0, 1), ints(dev, 41 + step), table, 1, grid(dev, 40 + step, 1))
        # the same row appended twice leaves what it left once
        assert torch.equal(stack.forward(y.clone(), batch=one), run_layers(stack, y.clone(), one))


@pytest.mark.parametrize('tokens,chunk', [(100, 64), (70, 32), (90, 50)])
def test_stack_chunked_prefill(dev, stack, tokens, chunk):
    """Overlapped chunks, which may end inside a block of scales, give what the chunks give one after
    another, bit for bit, with the same cache behind them."""
    batch = Batch(ints(dev, 0, tokens), ints(dev, tokens), ints(dev, [5, 0, 2, 7, 1, 4, 6]), None,
                  grid(dev, 0, tokens))
    x = prompt(dev, tokens, tokens)
    state = lambda: [t.clone() for b in stack.attention.values()
                     for t in (b.k_pages.view(torch.uint8), b.v_pages.view(torch.uint8), b.scales)]
    for b in stack.attention.values():
        b.allocate(8, 16, E4M3)
        b.k_pages.view(torch.uint8).zero_(), b.v_pages.view(torch.uint8).zero_()
    want = stack.prefill(x, chunk, overlap=False, batch=batch)
    pages = state()
    for b in stack.attention.values():
        b.k_pages.view(torch.uint8).zero_(), b.v_pages.view(torch.uint8).zero_(), b.scales.zero_()
    got = stack.prefill(x, chunk, batch=batch)
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    assert all(torch.equal(a, b) for a, b in zip(state(), pages))
    other = batch._replace(positions=grid(dev, 500, tokens))
    assert not torch.equal(stack.prefill(x, chunk, batch=other), want)  # the positions count


def test_stack_decode_graph(dev, stack):
    """A captured decode step of three sequences follows their lengths and positions between
    replays."""
    table = ints(dev, [0, 1], [2, 3], [4, 5])
    lengths, positions = ints(dev, 3, 17, 9), grid(dev, 0, 3)
    batch = Batch(ints(dev, 0, 1, 2, 3), lengths, table, 1, positions)
    for b in stack.attention.values():
        b.k_pages.copy_(torch.randn(b.k_pages.shape, device=dev).to(E4M3))
        b.v_pages.copy_(torch.randn(b.k_pages.shape, device=dev).to(E4M3))
        b.scales.fill_(0.5)
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
        lengths += 1
        positions += 1
        h = prompt(dev, 3, 20 + step)
        static.copy_(h)
        graph.replay()
        torch.cuda.synchronize()
        got = static.clone()
        # the eager step appends the same rows to the same places
        assert torch.equal(stack.forward(h.clone(), batch=batch), got)
