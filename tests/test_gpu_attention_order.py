"""GPU tests of attention calls in which single tokens behind many keys go before the prompts beside
them, over caches of 16 and 8 bits, against 64-bit results."""
import pytest
import torch

from tests.test_gpu_attention import attend as attend16
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
