"""CPU check of the attention block's rows: what forward_ refuses with W8A8 projections is what it
refuses with the others, before anything is launched."""
import pytest
import torch

from tests.test_attention_block_checks import H, batch, block, calls  # noqa: F401
from tests.test_attention_checks import gpu
from tests.test_block8_checks import pages


@pytest.mark.parametrize('w8a8', [False, True])
@pytest.mark.parametrize('dtype', [torch.float16, torch.float32])
def test_rows_of_other_types_are_refused(calls, dtype, w8a8):  # noqa: F811
    b = pages(block(w8a8=w8a8))
    for run in (b.check, b.forward_):
        with pytest.raises(ValueError):
            run(gpu(5, H, dtype=dtype), batch())
    assert not calls
