"""GPU tests of attention calls in which single tokens behind many keys go before the prompts beside
them, over caches of 16 and 8 bits, against 64-bit results."""
import pytest
import torch

from localmoe35ba3b_amd.operators import attention as A
from tests import cache8_util as C
from tests.conftest import seeded
from tests.test_gpu_attention import attend as attend16
from tests.test_gpu_attention import rand, to
from tests.test_gpu_cache8 import attend as attend8

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('call', [attend16, attend8])
@pytest.mark.parametrize('dim', [64, 128])
@pytest.mark.parametrize('sequences,keys,prompts', [
    (12, 4000, [(20, 20)]),  # far more bytes of single tokens' keys than tiles are worth
    (30, 900, [(40, 40), (17, 30), (130, 130)]),
    (30, 900, [(40, 900), (300, 700)]),  # about as many: in turn
    (90, 300, [(25, 25), (60, 61)])])  # more sequences than a wave looks at together
def test_many_single_tokens_beside_prompts(dev, call, dim, sequences, keys, prompts):
    gen = torch.Generator().manual_seed(sequences)
    length = torch.randint(keys // 2, keys * 3 // 2, (sequences,), generator=gen).tolist()
    lens = [(1, n) for n in length]
    for i, p in enumerate(prompts):  # among them, and a sequence without a new token
        lens.insert(7 * i + 3, p)
    lens.insert(5, (0, 50))
    call(dev, lens, 16, 8, 2, dim, torch.bfloat16, gate=True, pad=2, seed=dim)


@pytest.mark.parametrize('eight', [False, True])
@pytest.mark.parametrize('dim', [64, 128])
def test_captured_call_whose_order_changes(dev, dim, eight):
    """One captured call, replayed for batches of which some have single tokens first and others both in
    turn: bit for bit as in a call of its own, with eager work between the replays."""
    gen, page, pages = seeded(dim), 16, 600
    kp, vp, scales = C.random_cache(gen, pages, 2, page, dim, torch.bfloat16)
    if not eight:
        kp, vp = rand(gen, pages, 2, page, dim), rand(gen, pages, 2, page, dim)
    kp, vp, q = to(dev, kp, vp, rand(gen, 400, 8, dim))
    scales = scales.to(dev) if eight else None
    table = torch.randint(0, pages, (14, 200), generator=gen).to(torch.int32).to(dev)
    starts, lengths = (torch.zeros(n, dtype=torch.int32, device=dev) for n in (15, 14))
    out = torch.zeros_like(q)

    def call(o):
        return A.paged_attention(q, kp, vp, starts, lengths, table, out=o, scales=scales)

    call(out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out)
    first = [(1, 3000 - 100 * i) for i in range(11)] + [(30, 30), (17, 40), (0, 9)]
    turns = [(1, 300 - 10 * i) for i in range(11)] + [(300, 3000), (40, 900), (20, 20)]
    for lens in (first, turns, first[::-1], [(1, 3000)] * 14, turns[::-1], first):
        starts.copy_(torch.tensor([0] + [n for n, _ in lens]).cumsum(0))
        lengths.copy_(torch.tensor([n for _, n in lens]))
        out.fill_(3.0)
        graph.replay()
        want = call(torch.full_like(q, 3.0))
        torch.cuda.synchronize()
        assert torch.equal(out, want), lens
        assert out.isfinite().all() and (out[int(starts[-1]):] == 3.0).all()
