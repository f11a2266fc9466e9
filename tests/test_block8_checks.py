"""CPU checks of the attention block with a cache in 8 bits, positions of several axes and W8A8
projections: what it calls, and what is refused before anything is launched."""
import pytest
import torch

from localmoe35ba3b_amd.runtime.attention import AttentionBlock
from localmoe35ba3b_amd.runtime.stack import MoEStack
from tests.test_attention_block_checks import F32, H, I32, batch, block, calls  # noqa: F401
from tests.test_attention_checks import I64, gpu

E4M3 = torch.float8_e4m3fn


def pages(b, **change):
    b.k_pages, b.v_pages = (gpu(3, 2, 32, 64).to(E4M3) for _ in range(2))
    b.scales = gpu(3, 2, 2, 2, dtype=F32)
    for name, x in change.items():
        setattr(b, name, x)
    return b


def axes_block(**change):
    return pages(block(inv_freq=gpu(32, dtype=F32), axes=gpu(32, dtype=I32), **change))


def test_allocate():
    b = block().allocate(3, 32, E4M3)
    assert b.k_pages.dtype == b.v_pages.dtype == E4M3 and b.scales.shape == (3, 2, 2, 2)
    assert not b.scales.any()
    assert b.allocate(3, 32).scales is None and b.k_pages.dtype == torch.bfloat16


def test_what_a_block_calls(calls):  # noqa: F811
    h, p = gpu(5, H), batch(positions=gpu(3, 5, dtype=I64))
    b = axes_block()
    b.check(h, p)
    b.forward_(h, p)
    assert calls == ['lm_rmsnorm', 'lm_w8a16_linear', 'lm_paged_append_e4m3',
                     'lm_paged_attention_e4m3', 'lm_w8a16_linear']
    calls.clear()
    b = axes_block(w8a8=True)
    b.forward_(h, p)
    assert calls[:2] == ['lm_norm_quant_g128', 'lm_w8a8_gemm'] and calls[2:4] == [
        'lm_paged_append_e4m3', 'lm_paged_attention_e4m3'] and calls[4:] == ['lm_w8a8_linear']
    calls.clear()
    pages(block(), k_pages=gpu(3, 2, 16, 64), v_pages=gpu(3, 2, 16, 64), scales=None).forward_(
        h, batch(positions=gpu(5, dtype=I64)))
    assert calls[2:4] == ['lm_paged_append_axes', 'lm_paged_attention']


@pytest.mark.parametrize('change,message', [
    (dict(axes=gpu(32, dtype=I32)), 'axis'),  # no rotation
    (dict(axes=gpu(31, dtype=I32), inv_freq=gpu(32, dtype=F32)), 'axis')])
def test_blocks_that_could_not_run_are_refused(change, message):
    with pytest.raises(ValueError, match=message):
        block(**change)


def test_wide_rows_of_w8a8_are_refused():
    wide = 16512
    qkv = {'q': gpu(512, wide, dtype=torch.int8), 'scale': gpu(512, wide // 128, dtype=F32)}
    o = {'q': gpu(wide, 256, dtype=torch.int8), 'scale': gpu(wide, 2, dtype=F32)}
    AttentionBlock(qkv, o, 4, 2, 64, gated=False)
    with pytest.raises(ValueError, match='16384'):
        AttentionBlock(qkv, o, 4, 2, 64, gated=False, w8a8=True)


@pytest.mark.parametrize('positions', [None, gpu(3, 4, dtype=I64), gpu(3, 5, dtype=F32),
                                       gpu(2, 3, 5, dtype=I64)])
@pytest.mark.parametrize('w8a8', [False, True])
def test_positions_are_refused_before_the_append(calls, positions, w8a8):  # noqa: F811
    b = axes_block(w8a8=w8a8)
    for run in (b.check, b.forward_):
        with pytest.raises(ValueError, match='positions|position of every'):
            run(gpu(5, H), batch(positions=positions))
    assert not any('append' in c for c in calls)
    with pytest.raises(ValueError, match='axis of every pair'):  # no axes for several
        pages(block(inv_freq=gpu(32, dtype=F32))).check(gpu(5, H), batch(positions=gpu(3, 5, dtype=I64)))


@pytest.mark.parametrize('change,message', [
    (dict(scales=None), '8 bits'), (dict(scales=gpu(3, 2, 2, 1, dtype=F32)), 'scales'),
    (dict(k_pages=gpu(3, 2, 32, 64), v_pages=gpu(3, 2, 32, 64)), '8 bits')])
def test_caches_that_do_not_fit_are_refused(calls, change, message):  # noqa: F811
    b = pages(block(), **change)
    for run in (b.check, b.forward_):
        with pytest.raises(ValueError, match=message):
            run(gpu(5, H), batch())
    assert not any('append' in c for c in calls)


def test_chunks_take_their_part_of_the_positions():
    p = torch.arange(300).view(3, 100)
    b = batch(starts=torch.tensor([0, 100], dtype=I32), lengths=torch.tensor([130], dtype=I32),
              positions=p)
    parts = MoEStack._chunk_batches(None, b, 100, 64)
    assert torch.equal(parts[0].positions, p[:, :64]) and torch.equal(parts[1].positions, p[:, 64:])
    parts = MoEStack._chunk_batches(None, b._replace(positions=p[0]), 100, 64)
    assert torch.equal(parts[1].positions, p[0, 64:])
    assert MoEStack._chunk_batches(None, b._replace(positions=None), 100, 64)[1].positions is None
