"""GPU tests of w8a8.norm_quantize with rows that are added to themselves, in every form of its kernel."""
import pytest
import torch

from localmoe35ba3b_amd.operators import w8a8
from tests.conftest import seeded
from tests.test_gpu_norm_quantize import TYPES, check, rows

pytestmark = pytest.mark.gpu


@TYPES
@pytest.mark.parametrize('n,k', [(5, 256), (5, 512), (3, 640), (300, 2048), (7, 2176), (33, 4096), (3, 4224),
                                 (33, 8192), (2, 8320), (33, 16384)])
def test_rows_added_to_themselves(dev, n, k, dtype):
    """The same bits as with a copy of the rows, and the norm of the doubled rows."""
    gen = seeded(n * k)
    h = rows(gen, n, k, dtype)
    weight = torch.randn(k, generator=gen) * 0.2
    one, two = h.to(dev), h.to(dev)
    q, s = w8a8.norm_quantize(one, weight.to(dev), add=one)
    q2, s2 = w8a8.norm_quantize(two, weight.to(dev), add=two.clone())
    assert torch.equal(one.cpu(), h * 2) and torch.equal(two, one)
    assert torch.equal(q, q2) and torch.equal(s, s2)
    check(q, s, h * 2, weight)
