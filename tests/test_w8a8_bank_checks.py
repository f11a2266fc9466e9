"""CPU checks of the W8A8 products' weights and scales: what a kernel would read as something else, or
not at all, is refused before a launch, by the operators and by the attention block."""
import pytest
import torch

from localmoe35ba3b_amd import _lib
from localmoe35ba3b_amd.operators import w8a8
from localmoe35ba3b_amd.runtime.attention import AttentionBlock
from tests.test_attention_checks import F32, gpu

I8 = torch.int8


def linear(rows=5, **change):
    a = dict(x=gpu(rows, 256), q=gpu(32, 256, dtype=I8), scale=gpu(32, 2, dtype=F32))
    a.update(change)
    return w8a8.linear(**a)


def gemm(**change):
    a = dict(xq=gpu(5, 256, dtype=I8), xs=gpu(5, 2, dtype=F32), q=gpu(32, 256, dtype=I8),
             scale=gpu(32, 2, dtype=F32))
    a.update(change)
    return w8a8.gemm(**a)


@pytest.mark.parametrize('run,change', [
    (linear, dict(scale=gpu(32, 2))), (linear, dict(scale=torch.zeros(32, 2))),
    (linear, dict(q=gpu(32, 256))), (linear, dict(q=torch.zeros(32, 256, dtype=I8))),
    (linear, dict(rows=20, scale=gpu(32, 2))), (linear, dict(rows=20, q=gpu(32, 256))),
    (gemm, dict(scale=gpu(32, 2))), (gemm, dict(scale=torch.zeros(32, 2))),
    (gemm, dict(xs=gpu(5, 2))), (gemm, dict(xs=torch.zeros(5, 2))), (gemm, dict(q=gpu(32, 256)))])
def test_operators_refuse_other_banks(run, change, monkeypatch):
    calls = []
    monkeypatch.setattr(_lib, 'call', lambda name, *args: calls.append(name))
    monkeypatch.setattr(_lib, 'stream', lambda device=None: 0)
    run(**{n: v for n, v in change.items() if n == 'rows'})
    assert calls
    at = len(calls)
    with pytest.raises(ValueError):
        run(**change)
    assert not any('gemm' in c or 'linear' in c for c in calls[at:])


@pytest.mark.parametrize('w8a8', [False, True])
@pytest.mark.parametrize('side,name,dtype', [('qkv', 'q', torch.uint8), ('qkv', 'scale', torch.bfloat16),
                                             ('o', 'q', torch.uint8), ('o', 'scale', torch.float16)])
def test_blocks_refuse_other_banks(side, name, dtype, w8a8):
    banks = dict(qkv={'q': gpu(512, 256, dtype=I8), 'scale': gpu(512, 2, dtype=F32)},
                 o={'q': gpu(256, 256, dtype=I8), 'scale': gpu(256, 2, dtype=F32)})
    AttentionBlock(**banks, q_heads=4, kv_heads=2, head_dim=64, gated=False, w8a8=w8a8)
    banks[side][name] = gpu(*banks[side][name].shape, dtype=dtype)
    with pytest.raises(ValueError, match='int8 projections'):
        AttentionBlock(**banks, q_heads=4, kv_heads=2, head_dim=64, gated=False, w8a8=w8a8)
    banks[side][name] = torch.empty(banks[side][name].shape, device='meta',
                                    dtype=I8 if name == 'q' else F32)  # stands for another device
    with pytest.raises(ValueError, match='one device'):
        AttentionBlock(**banks, q_heads=4, kv_heads=2, head_dim=64, gated=False, w8a8=w8a8)


def test_blocks_refuse_rows_wider_than_their_second_product():
    heads = 1028  # 65792 channels
    banks = dict(qkv={'q': gpu(heads * 64 * 3, 128, dtype=I8), 'scale': gpu(heads * 64 * 3, 1, dtype=F32)},
                 o={'q': gpu(128, heads * 64, dtype=I8), 'scale': gpu(128, heads // 2, dtype=F32)})
    AttentionBlock(**banks, q_heads=heads, kv_heads=heads, head_dim=64, gated=False)
    with pytest.raises(ValueError, match='65536'):
        AttentionBlock(**banks, q_heads=heads, kv_heads=heads, head_dim=64, gated=False, w8a8=True)
