"""GPU tests of w8a8.norm_quantize against 64-bit results: the residual's addition, the norm and the
8-bit rows, alone and on their way through the W8A8 product."""
import math

import pytest
import torch

from localmoe35ba3b_amd import router
from localmoe35ba3b_amd.operators import w8a8
from tests.conftest import seeded

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16
TYPES = pytest.mark.parametrize('dtype', [BF16, FP16])
EPS = 1e-6


def rows(gen, n, k, dtype, scale=1.0):
    x = torch.randn(n, k, generator=gen) * scale
    x[:, torch.randint(k, (3,), generator=gen)] *= 40.0  # strong channels
    return x.to(dtype)


def check(q, s, h, weight, what=''):
    """q and s against the norm of the rows h in 64 bits."""
    n, k = h.shape
    h = h.double()
    m = h / torch.sqrt(h.square().mean(-1, keepdim=True) + EPS)
    if weight is not None:
        m = m * (1 + weight.double())
    m = m.view(n, k // 128, 128)
    # fp32: the sum of squares (of one sign, k additions and products at most, half of it under the
    # root), the mean, eps, root and quotient, two products and 1 + w
    err = (k + 8) * 2.0 ** -24
    amax = m.abs().amax(-1)
    want = torch.clamp(amax, min=1e-10) / 127
    s, q = s.cpu().double(), q.cpu().double().view(m.shape)
    assert ((s - want).abs() <= want * (err + 3 * 2.0 ** -24)).all(), what  # two products more
    # half a step, what m is off by, and the quotient's rounding of at most 127 steps
    off = (q * s[..., None] - m).abs()
    assert (off <= s[..., None] * (0.5 + 127 * 2.0 ** -23) + m.abs() * err).all(), what
    assert q.abs().max() <= 127
    assert (q.abs().amax(-1)[amax > 1e-9] == 127).all(), what


@TYPES
@pytest.mark.parametrize('add', [False, True])
@pytest.mark.parametrize('n,k', [(1, 128), (3, 256), (1, 2048), (5, 640), (257, 2048), (2, 2176),
                                 (7, 4096), (3, 4224), (2, 8192), (3, 8320), (2, 16384)])
def test_norm_quantize(dev, n, k, add, dtype):
    gen = seeded(n + k)
    h, x = rows(gen, n, k, dtype, 3.0), rows(gen, n, k, dtype)
    weight = torch.randn(k, generator=gen) * 0.2 if k % 256 else None
    hd = h.to(dev)
    before = hd.clone()
    q, s = w8a8.norm_quantize(hd, None if weight is None else weight.to(dev), EPS,
                              add=x.to(dev) if add else None)
    assert q.shape == (n, k) and q.dtype == torch.int8 and s.shape == (n, k // 128)
    if add:
        h = (h.float() + x.float()).to(dtype)
        assert torch.equal(hd.cpu(), h)
    else:
        assert torch.equal(hd, before)
    check(q, s, h, weight)


@TYPES
def test_rows_of_zeros_and_of_far_sizes(dev, dtype):
    """Zero rows (scales of the least value), tiny and large ones, a group of zeros in a row."""
    gen = seeded(2)
    h = torch.randn(6, 512, generator=gen)
    h[0] = 0
    h[1] *= 1e-4
    h[2] *= 200.0
    h[3, 128:256] = 0
    h[4, 1:] = 0
    h = h.to(dtype)
    q, s = w8a8.norm_quantize(h.to(dev))
    check(q, s, h, None)
    assert not q[0].any() and not q[3, 128:256].any()
    a, b = w8a8.norm_quantize(h.to(dev), add=-h.to(dev))
    assert not a.any() and torch.equal(b, torch.full_like(b, 1e-10) * (1.0 / 127.0))


def test_not_finite_rows_show_in_their_scales(dev):
    """Infinities and NaN leave scales that are not finite, in their rows only."""
    h = torch.randn(4, 256, generator=seeded(3)).to(BF16)
    h[1, 7], h[2, 200] = math.nan, math.inf
    q, s = w8a8.norm_quantize(h.to(dev))
    values = q.cpu().double().view(4, 2, 128) * s.cpu().double()[..., None]
    assert not values[1].isfinite().any() and not values[2, 1].isfinite().all()
    check(q[[0, 3]], s[[0, 3]], h[[0, 3]], None)


def test_layouts_and_refusals(dev):
    """Rows to add with a pitch, themselves, on another stream; h of a pitch only without them."""
    gen = seeded(4)
    h, x = rows(gen, 9, 256, BF16).to(dev), rows(gen, 9, 300, BF16).to(dev)
    want_h = (h.float() + x[:, 3:259].float()).to(BF16)
    got = h.clone()
    q, s = w8a8.norm_quantize(got, add=x[:, 3:259])
    assert torch.equal(got, want_h)
    wide = torch.zeros(9, 300, dtype=BF16, device=dev)
    wide[:, 1:257] = got
    again = w8a8.norm_quantize(wide[:, 1:257])
    assert torch.equal(again[0], q) and torch.equal(again[1], s)
    with pytest.raises(ValueError, match='contiguous'):
        w8a8.norm_quantize(wide[:, 1:257], add=h)
    twice = h.clone()
    w8a8.norm_quantize(twice, add=twice)
    assert torch.equal(twice, h * 2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    other = h.clone()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        q2, s2 = w8a8.norm_quantize(other, add=x[:, 3:259])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(q2, q) and torch.equal(s2, s) and torch.equal(other, want_h)
    q, s = w8a8.norm_quantize(h[:0])
    assert q.shape == (0, 256) and s.shape == (0, 2)


def test_against_the_separate_operators(dev):
    """router.rmsnorm and quantize round the normed row to bf16 in between: the values agree within
    that rounding (2^-8 of a value, and of the group's largest in its scale) and a step."""
    h = rows(seeded(5), 33, 2048, BF16).to(dev)
    w = torch.randn(2048, generator=seeded(6)).to(dev) * 0.1
    q, s = w8a8.norm_quantize(h, w)
    q0, s0 = w8a8.quantize(router.rmsnorm(h, w))
    a, b = ((x.double().view(33, 16, 128) * y.double()[..., None]) for x, y in ((q, s), (q0, s0)))
    assert ((a - b).abs() <= (s + s0)[..., None] * 0.51 + 2.0 ** -8 * 1.01 * a.abs().amax(-1, keepdim=True)).all()


def test_captured_with_its_product(dev):
    """norm_quantize and gemm in a graph, replayed while the rows change, with eager work between."""
    gen = seeded(7)
    wq = torch.randint(-127, 128, (640, 2048), generator=gen, dtype=torch.int8).to(dev)
    ws = (torch.rand(640, 16, generator=gen) * 1e-3).to(dev)
    h, x = rows(gen, 40, 2048, BF16).to(dev), rows(gen, 40, 2048, BF16).to(dev)

    def run(h):
        q, s = w8a8.norm_quantize(h, add=x)
        return w8a8.gemm(q, s, wq, ws)

    run(h.clone())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(h)
    for _ in range(4):
        h.copy_(rows(gen, 40, 2048, BF16))
        x.copy_(rows(gen, 40, 2048, BF16))
        eager = h.clone()
        want = run(eager)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(h, eager)
