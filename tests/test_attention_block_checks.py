"""CPU checks of the attention block and of the norm before it: what is refused before
anything is launched."""
import pytest
import torch

from localmoe35ba3b_amd import _lib, router
from localmoe35ba3b_amd.runtime.attention import AttentionBlock, Batch
from tests.test_attention_checks import gpu

F32, I32, FP16, H = torch.float32, torch.int32, torch.float16, 256


@pytest.fixture
def calls(monkeypatch):
    """The names of the entry points that are called; nothing is launched."""
    got = []
    monkeypatch.setattr(_lib, 'call', lambda name, *args: got.append(name))
    monkeypatch.setattr(_lib, 'launch', lambda device, name, *args: got.append(name))
    monkeypatch.setattr(_lib, 'stream', lambda device=None: 0)
    return got


def block(**change):
    a = dict(q_heads=4, kv_heads=2, head_dim=64, gated=False)
    a.update(change)
    rows = (a['q_heads'] * (2 if a['gated'] else 1) + 2 * a['kv_heads']) * a['head_dim']
    wide = a['q_heads'] * a['head_dim']
    qkv = {'q': gpu(rows, H, dtype=torch.int8), 'scale': gpu(rows, H // 128, dtype=F32)}
    o = {'q': gpu(H, wide, dtype=torch.int8), 'scale': gpu(H, wide // 128, dtype=F32)}
    return AttentionBlock(qkv, o, **a)


def pages(b, dtype=torch.bfloat16):
    b.k_pages, b.v_pages = gpu(3, 2, 16, 64, dtype=dtype), gpu(3, 2, 16, 64, dtype=dtype)
    return b


def batch(**change):
    a = dict(starts=gpu(2, dtype=I32), lengths=gpu(1, dtype=I32), table=gpu(1, 3, dtype=I32))
    a.update(change)
    return Batch(**a)


@pytest.mark.parametrize('x,weight', [
    (gpu(5, H, dtype=FP16), None), (gpu(5, H, dtype=F32), None),
    (torch.zeros(5, H, dtype=torch.bfloat16), None),
    (gpu(5, H), gpu(H - 1, dtype=F32)), (gpu(5, H), gpu(2 * H, dtype=F32))])
def test_rmsnorm_refusals(calls, x, weight):
    """Rows of other types would be read as bf16, host memory and weights that are too short by
    the GPU."""
    router.rmsnorm(gpu(5, H), gpu(H, dtype=F32))
    router.rmsnorm(gpu(5, H))
    assert calls == ['lm_rmsnorm'] * 2
    with pytest.raises(ValueError, match='rows'):
        router.rmsnorm(x, weight)
    assert len(calls) == 2


@pytest.mark.parametrize('h', [gpu(5, H, dtype=FP16), torch.zeros(5, H, dtype=torch.bfloat16)])
@pytest.mark.parametrize('dtype', [torch.bfloat16, FP16])
def test_block_refuses_rows_that_its_norm_cannot_read(calls, h, dtype):
    b = pages(block(), dtype)
    with pytest.raises(ValueError, match='bf16'):
        b.forward_(h, batch())
    assert not calls


@pytest.mark.parametrize('dtype', [FP16, F32])
def test_allocate_refuses_types_that_the_block_never_writes(dtype):
    """The block's rows are bf16, so are the keys and values it appends."""
    with pytest.raises(ValueError, match='bf16'):
        block().allocate(3, 16, dtype=dtype)
    with pytest.raises(ValueError, match='bf16'):
        block().allocate(3, 16, dtype)


@pytest.mark.parametrize('size', [0, 8, 24, 2048])
def test_allocate_refuses_pages_that_the_operators_do(size):
    with pytest.raises(ValueError, match='page size'):
        block().allocate(3, size)


def test_allocate():
    b = block().allocate(3, 16, torch.bfloat16)
    assert b.k_pages.shape == b.v_pages.shape == (3, 2, 16, 64)
    assert b.k_pages.dtype == b.v_pages.dtype == torch.bfloat16
    assert block().allocate(2).k_pages.shape == (2, 2, 64, 64)


@pytest.mark.parametrize('change,message', [
    (dict(q_heads=3), 'heads'), (dict(head_dim=32, q_heads=8), 'heads of'),
    (dict(norm=gpu(H + 1, dtype=F32)), 'norm'), (dict(q_norm=gpu(32, dtype=F32)), 'norm'),
    (dict(k_norm=gpu(65, dtype=F32)), 'norm'), (dict(inv_freq=gpu(12, dtype=F32)), 'multiple of 16'),
    (dict(inv_freq=gpu(40, dtype=F32)), 'multiple of 16')])
def test_blocks_that_could_not_run_are_refused(change, message):
    """What the operators would refuse in every step."""
    block(norm=gpu(H, dtype=F32), q_norm=gpu(64, dtype=F32), k_norm=gpu(64, dtype=F32),
          inv_freq=gpu(32, dtype=F32))
    with pytest.raises(ValueError, match=message):
        block(**change)


def test_projections_without_their_scales_are_refused():
    a = block()
    for name in ('qkv', 'o'):
        bank = {'q': getattr(a, name)['q'], 'scale': getattr(a, name)['scale'][:, :1]}
        pair = {'qkv': a.qkv, 'o': a.o, name: bank}
        with pytest.raises(ValueError, match='scales'):
            AttentionBlock(pair['qkv'], pair['o'], 4, 2, 64, gated=False)


@pytest.mark.parametrize('h', [gpu(1, 5, H), gpu(5, H + 128), gpu(H)])
def test_block_refuses_other_rows(calls, h):
    for run in (pages(block()).forward_, pages(block()).check):
        with pytest.raises(ValueError):
            run(h, batch())
    assert 'lm_paged_append' not in calls


@pytest.mark.parametrize('change', [dict(max_new=-1), dict(starts=gpu(2, dtype=torch.int64)),
                                    dict(table=gpu(2, 3, dtype=I32))])
def test_block_refuses_batches_before_it_appends(calls, change):
    b = pages(block())
    with pytest.raises(ValueError):
        b.forward_(gpu(5, H), batch(**change))
    assert 'lm_paged_append' not in calls
    calls.clear()
    b.forward_(gpu(5, H), batch())
    assert calls == ['lm_rmsnorm', 'lm_w8a16_linear', 'lm_paged_append', 'lm_paged_attention',
                     'lm_w8a16_linear']


def test_projections_that_int8_linear_refuses():
    """One head of 64 channels leaves the output projection half a group of 128."""
    with pytest.raises(ValueError, match='128'):
        block(q_heads=1, kv_heads=1)


@pytest.mark.parametrize('heads', [dict(q_heads=0), dict(q_heads=2, kv_heads=0)])
def test_blocks_without_heads_are_refused(heads):
    with pytest.raises(ValueError, match='heads'):
        block(**heads)
