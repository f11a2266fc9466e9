"""CPU checks of the operators on a cache in 8 bits, of positions with several axes and of
norm_quantize: what is refused before a launch, by Python and by the C entry points, and what reaches
the library."""
import pytest
import torch

from localmoe35ba3b_amd import _lib
from localmoe35ba3b_amd.operators import attention as A
from localmoe35ba3b_amd.operators import w8a8
from tests.test_attention_checks import F32, I32, I64, batch, calls, gpu  # noqa: F401

E4M3, BF16 = torch.float8_e4m3fn, torch.bfloat16


def norm(**change):
    a = dict(q=gpu(5, 4, 128), k=gpu(5, 2, 128), q_weight=None, k_weight=None,
             positions=gpu(3, 5, dtype=I64), inv_freq=gpu(32, dtype=F32), axes=gpu(32, dtype=I32))
    a.update(change)
    return A.qk_norm_rope(**a)


def batch8(**change):
    return batch(**{**dict(k_pages=gpu(6, 2, 32, 128).to(E4M3), v_pages=gpu(6, 2, 32, 128).to(E4M3),
                           scales=gpu(6, 2, 2, 2, dtype=F32)), **change})


def append(**change):
    return A.append(**batch8(**{**dict(k=gpu(5, 2, 128), v=gpu(5, 2, 128), q=gpu(5, 4, 128),
                                       inv_freq=gpu(32, dtype=F32)), **change}))


def attend(**change):
    return A.paged_attention(**batch8(**{**dict(q=gpu(5, 4, 128)), **change}))


def normq(**change):
    a = dict(h=gpu(5, 256), weight=gpu(256, dtype=F32), add=gpu(5, 256))
    a.update(change)
    return w8a8.norm_quantize(**a)


REFUSED = [
    (norm, dict(axes=None), 'axis of every pair'), (norm, dict(axes=gpu(31, dtype=I32)), 'axis'),
    (norm, dict(positions=gpu(3, 4, dtype=I64)), 'position'),
    (norm, dict(positions=gpu(3, 5, dtype=F32)), 'whole positions'),
    (norm, dict(positions=gpu(65, 5, dtype=I64)), 'axes of positions'),
    (norm, dict(positions=gpu(0, 5, dtype=I64)), 'axes of positions'),
    (norm, dict(positions=gpu(1, 3, 5, dtype=I64)), 'position'),
    (append, dict(axes=gpu(32, dtype=I32)), 'positions'),
    (append, dict(positions=gpu(3, 5, dtype=I64)), 'axis of every pair'),
    (append, dict(positions=gpu(4, dtype=I64)), 'position'),
    (append, dict(positions=gpu(5, dtype=I64), axes=gpu(30, dtype=I32)), 'axis'),
    (append, dict(scales=None), '8 bits'), (attend, dict(scales=None), '8 bits'),
    (append, dict(k_pages=gpu(6, 2, 32, 128), v_pages=gpu(6, 2, 32, 128)), '8 bits'),
    (attend, dict(k_pages=gpu(6, 2, 32, 128), v_pages=gpu(6, 2, 32, 128)), '8 bits'),
    (attend, dict(v_pages=gpu(6, 2, 32, 128)), '8 bits'),
    (attend, dict(q=gpu(5, 4, 128, dtype=F32)), 'FP16/BF16'),
    (append, dict(scales=gpu(6, 2, 2, 1, dtype=F32)), 'scales'),
    (attend, dict(scales=gpu(6, 2, 2, 2, dtype=BF16)), 'scales'),
    (attend, dict(scales=gpu(6, 2, 4, dtype=F32)), 'scales'),
    (attend, dict(scales=gpu(6, 2, 2, 4, dtype=F32)[..., ::2]), 'contiguous'),
    (append, dict(scales=gpu(6, 2, 2, 2, dtype=F32).transpose(1, 2)), 'contiguous'),
    (normq, dict(h=gpu(5, 200), add=None, weight=None), 'multiple of 128'),
    (normq, dict(h=gpu(5, 16512), add=None, weight=None), '16384'),
    (normq, dict(h=gpu(5, 0), add=None, weight=None), '128'),
    (normq, dict(h=gpu(5, 256, dtype=F32)), 'CUDA rows'), (normq, dict(h=gpu(5, 2, 256)), 'CUDA rows'),
    (normq, dict(h=torch.zeros(5, 256, dtype=BF16)), 'CUDA rows'),
    (normq, dict(weight=gpu(128, dtype=F32)), 'norm weight'),
    (normq, dict(add=gpu(4, 256)), 'match'), (normq, dict(add=gpu(5, 256, dtype=torch.float16)), 'match'),
    (normq, dict(h=gpu(5, 512)[:, ::2]), 'contiguous'),
    (normq, dict(h=gpu(5 * 256 + 8)[1:1281].view(5, 256)), 'contiguous'),
]


@pytest.mark.parametrize('run,change,message', REFUSED)
def test_refusals(calls, run, change, message):  # noqa: F811
    run()
    assert len(calls) == 1
    with pytest.raises(ValueError, match=message):
        run(**change)
    assert len(calls) == 1


def test_what_reaches_the_library(calls):  # noqa: F811
    """The entry point of each form, and the arguments that only it has."""
    norm()
    norm(positions=gpu(5, dtype=I64), axes=None)
    norm(positions=gpu(1, 5, dtype=I64), axes=None)
    assert [c[0] for c in calls] == ['lm_qk_norm_rope_axes', 'lm_qk_norm_rope', 'lm_qk_norm_rope']
    assert calls[0][1][13:15] == (5, 3)
    del calls[:]
    append()
    append(positions=gpu(3, 5, dtype=I64), axes=gpu(32, dtype=I32))
    plain = dict(k_pages=gpu(6, 2, 32, 128), v_pages=gpu(6, 2, 32, 128), scales=None)
    append(**plain)
    append(**plain, positions=gpu(5, dtype=torch.int32))
    assert [c[0] for c in calls] == ['lm_paged_append_e4m3', 'lm_paged_append_e4m3',
                                     'lm_paged_append', 'lm_paged_append_axes']
    for (name, args), places in zip(calls, ((0, 0, 1, 0), (5, 3), None, (5, 1, 0))):
        if name == 'lm_paged_append_e4m3':
            assert args[16:21] == (8, 6, 2 * 32 * 128, 2, 32)
            assert args[28:32] == places if places[0] == 0 else args[29:31] == places
    assert calls[3][1][27:30] == (5, 1, 0)
    del calls[:]
    layers = gpu(6, 3, 2, 2, 2, dtype=F32)
    both = gpu(6, 2, 2, 32, 128).to(E4M3).as_subclass(type(layers))
    attend(scales=layers[:, 1], k_pages=both[:, 0], v_pages=both[:, 1])
    name, args = calls.pop()
    assert name == 'lm_paged_attention_e4m3'
    assert args[6:10] == (layers[:, 1].data_ptr(), 24, 6, 2 * 2 * 32 * 128)
    one = gpu(1, 2, 2, 2, dtype=F32)
    attend(scales=one, k_pages=both[:1, 0], v_pages=both[:1, 1])
    assert calls.pop()[1][7] == 8
    normq(add=gpu(5, 260)[:, :256])
    name, args = calls.pop()
    assert name == 'lm_norm_quant_g128' and args[5:7] == (5, 256) and args[1] % 16 == 0


def c_call(entry, **change):
    """A C call with placeholder pointers, refused before any use."""
    at = 4096
    a = dict(q=at, q_token=512, q_head=128, q_heads=4, q_w=None, q_out=at, k=at, k_token=256,
             k_head=128, k_heads=2, k_w=None, k_out=at, v=at, positions=at, position_stride=5, axes=3,
             axis=at, freq=at, pairs=32, tokens=5, dim=128, dtype=0, k_pages=at, v_pages=at,
             scales=at, scale_stride=4, pages=6, page_stride=4096, page=16, starts=at, lengths=at,
             table=at, table_stride=3, table_pages=3, sequences=2, max_new=5, gate=None, out=at, ws=at,
             ws_bytes=1 << 40, h=at, x=at, w=at, n=256, s=at)
    a.update(change)
    pick = lambda *names: [a[n] for n in names]
    cache = pick('pages', 'page_stride', 'k_heads', 'page', 'dim', 'starts', 'lengths', 'table',
                 'table_stride', 'table_pages', 'sequences')
    places = pick('positions', 'position_stride', 'axes', 'axis', 'freq', 'pairs', 'tokens')
    rows = pick('k', 'k_token', 'k_head', 'k_w', 'v', 'k_token', 'k_head', 'q', 'q_token', 'q_head',
                'q_heads', 'q_w', 'q_out', 'k_pages', 'v_pages')
    lib = _lib.lib()
    if entry == 'norm':
        rc = lib.lm_qk_norm_rope_axes(*pick('q', 'q_token', 'q_head', 'q_heads', 'q_w', 'q_out', 'k',
                                            'k_token', 'k_head', 'k_heads', 'k_w', 'k_out'), *places,
                                      a['dim'], 1e-6, a['dtype'], None)
    elif entry == 'append':
        rc = lib.lm_paged_append_axes(*rows, *cache, *places, 1e-6, a['dtype'], None)
    elif entry == 'append8':
        rc = lib.lm_paged_append_e4m3(*rows, a['scales'], a['scale_stride'], *cache, *places, 1e-6,
                                      a['dtype'], None)
    elif entry == 'attend8':
        rc = lib.lm_paged_attention_e4m3(
            *pick('q', 'q_token', 'q_head', 'q_heads', 'k_pages', 'v_pages', 'scales', 'scale_stride'),
            *cache, a['tokens'], a['max_new'], 0.1, a['gate'], 0, 0, a['out'], a['ws'], a['ws_bytes'],
            a['dtype'], None)
    else:
        rc = lib.lm_norm_quant_g128(*pick('h', 'x', 'w', 'q', 's', 'tokens', 'n'), 1e-6, a['dtype'],
                                    None)
    return rc, lib.lm_last_error().decode()


AXES, EIGHT = ('norm', 'append', 'append8'), ('append8', 'attend8')
C_REFUSED = [
    (AXES, dict(axes=0), 'axes'), (AXES, dict(axes=65), 'axes'), (AXES, dict(position_stride=4), 'overlap'),
    (AXES, dict(positions=None), 'positions'), (('norm',), dict(positions=None, axis=None), 'null'),
    (AXES + ('attend8',), dict(dtype=2), 'FP16/BF16'), (AXES + ('attend8',), dict(dim=96), 'heads of'),
    (AXES + ('attend8',), dict(q=4104), 'aligned'), (AXES, dict(pairs=12), 'multiple of 16'),
    (AXES + ('attend8',), dict(tokens=1 << 24), 'token count'),
    (EIGHT, dict(scales=None), 'scales'), (EIGHT, dict(scales=4098), 'scales'),
    (EIGHT, dict(scale_stride=3), 'scales'), (EIGHT, dict(scale_stride=-4), 'scales'),
    (EIGHT, dict(page_stride=4104), 'pages'), (EIGHT, dict(page_stride=4080), 'pages'),
    (EIGHT, dict(page=8), 'page size'), (EIGHT, dict(table_pages=1 << 27), 'page table'),
    (EIGHT, dict(k_pages=4104), 'aligned'), (EIGHT, dict(starts=None), 'null'),
    (('append8',), dict(v=None), 'aligned'), (('append8',), dict(q_out=None), 'aligned'),
    # a workgroup for each token and each block: 2^24 are refused, whatever the heads
    (('append8',), dict(tokens=(1 << 24) - 1, position_stride=1 << 24), 'too many rows'),
    (('attend8',), dict(q_heads=5), 'multiple'), (('attend8',), dict(out=4104), 'aligned'),
    (('attend8',), dict(ws=None), 'workspace'), (('attend8',), dict(ws=4104), 'workspace'),
    (('quant',), dict(n=100), 'multiple of 128'), (('quant',), dict(n=0), 'multiple of 128'),
    (('quant',), dict(n=16512), 'multiple of 128'), (('quant',), dict(dtype=2), 'CUDA rows'),
    (('quant',), dict(tokens=-1), 'rows'), (('quant',), dict(tokens=1 << 24), 'rows'),
    (('quant',), dict(h=None), 'null'), (('quant',), dict(s=None), 'null'),
    (('quant',), dict(h=4104), 'aligned'), (('quant',), dict(x=4104), 'aligned'),
    (('quant',), dict(w=4100), 'aligned'), (('quant',), dict(q=4100), 'aligned'),
]


@pytest.mark.parametrize('entry,change,message', [(e, c, m) for es, c, m in C_REFUSED for e in es])
def test_c_refusals(entry, change, message):
    rc, error = c_call(entry, **change)
    assert rc == _lib.LM_EINVAL and message in error


def test_c_workspace_is_large_enough():
    rc, error = c_call('attend8', ws_bytes=16)
    assert rc == _lib.LM_ENOMEM and 'too small' in error


@pytest.mark.parametrize('entry', AXES + ('attend8', 'quant'))
def test_c_calls_without_work(entry):
    """No tokens, and no sequences: nothing is launched and no pointer is used."""
    assert c_call(entry, tokens=0, q=None, k=None, h=None, scales=None)[0] == _lib.LM_OK
    if entry not in ('norm', 'quant'):
        assert c_call(entry, sequences=0, q=None, k=None, starts=None, scales=None)[0] == _lib.LM_OK
