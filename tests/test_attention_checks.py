"""CPU checks of the attention operators: what is refused before a launch, by the Python
operators and by the C entry points, and what reaches the library."""
import pytest
import torch

from localmoe35ba3b_amd import _lib
from localmoe35ba3b_amd.operators import attention as A


class OnGpu(torch.Tensor):
    """A tensor that claims to be on the GPU; it reaches the checks, nothing is launched."""
    is_cuda = True


def gpu(*shape, dtype=torch.bfloat16):
    """Zeros at a 16-byte aligned address."""
    t = torch.zeros(*shape, dtype=dtype)
    assert t.data_ptr() % 16 == 0
    return t.as_subclass(OnGpu)


@pytest.fixture
def calls(monkeypatch):
    got = []
    monkeypatch.setattr(_lib, 'launch', lambda device, name, *args: got.append((name, args)))
    return got


def norm(**change):
    a = dict(q=gpu(5, 4, 128), k=gpu(5, 2, 128), q_weight=gpu(128, dtype=torch.float32),
             k_weight=None, positions=gpu(5, dtype=torch.int64), inv_freq=gpu(32, dtype=torch.float32))
    a.update(change)
    return A.qk_norm_rope(**a)


def batch(**change):
    a = dict(k_pages=gpu(6, 2, 16, 128), v_pages=gpu(6, 2, 16, 128),
             starts=gpu(3, dtype=torch.int32), lengths=gpu(2, dtype=torch.int32),
             table=gpu(2, 3, dtype=torch.int32))
    a.update(change)
    return a


def append(**change):
    a = batch(k=gpu(5, 2, 128), v=gpu(5, 2, 128), q=gpu(5, 4, 128),
              inv_freq=gpu(32, dtype=torch.float32))
    a.update(change)
    return A.append(**a)


def attend(**change):
    a = batch(q=gpu(5, 4, 128))
    a.update(change)
    return A.paged_attention(**a)


F32, I32, I64 = torch.float32, torch.int32, torch.int64
REFUSED = [
    (norm, dict(q=torch.zeros(5, 4, 128, dtype=torch.bfloat16)), 'CUDA'),
    (norm, dict(q=gpu(5, 512)), 'heads, head_dim'),
    (norm, dict(q=gpu(5, 4, 128, dtype=F32)), 'FP16/BF16'),
    (norm, dict(k=gpu(5, 2, 128, dtype=torch.float16)), 'share'),
    (norm, dict(k=gpu(4, 2, 128)), 'match'),
    (norm, dict(k=gpu(5, 2, 64)), 'match'),
    (norm, dict(q_weight=gpu(64, dtype=F32)), 'norm weight'),
    (norm, dict(positions=gpu(4, dtype=I64)), 'position'),
    (norm, dict(inv_freq=gpu(12, dtype=F32)), 'multiple of 16'),
    (norm, dict(inv_freq=gpu(72, dtype=F32)), 'multiple of 16'),
    (norm, dict(inv_freq=gpu(0, dtype=F32)), 'multiple of 16'),
    (append, dict(k=gpu(5, 3, 128)), 'cache'),
    (append, dict(v=gpu(4, 2, 128)), 'cache'),
    (append, dict(v=gpu(5, 2, 128, dtype=torch.float16)), 'share'),
    (append, dict(q=gpu(4, 4, 128)), 'match'),
    (append, dict(v_pages=gpu(6, 2, 32, 128)), 'pages'),
    (append, dict(k_pages=gpu(6, 16, 2, 128).transpose(1, 2)), 'pages'),
    (append, dict(k_pages=gpu(6, 16, 2, 128).transpose(1, 2),
                  v_pages=gpu(6, 16, 2, 128).transpose(1, 2)), 'contiguous'),
    (append, dict(starts=gpu(3, dtype=I64)), 'int32'),
    (append, dict(starts=gpu(2, dtype=I32)), 'match'),
    (append, dict(table=gpu(3, 3, dtype=I32)), 'match'),
    (append, dict(table=gpu(6, dtype=I32)), 'match'),
    (append, dict(table=gpu(3, 2, dtype=I32).t()), 'contiguous'),
    (append, dict(lengths=gpu(4, dtype=I32)[::2]), 'contiguous'),
    (attend, dict(q=gpu(5, 3, 128)), 'cache'),
    (attend, dict(q=gpu(5, 4, 64)), 'cache'),
    (attend, dict(q=gpu(5, 4, 128, dtype=torch.float16)), 'share'),
    (attend, dict(gate=gpu(5, 2, 128)), 'gate'),
    (attend, dict(out=gpu(5, 2, 128)), 'output'),
    (attend, dict(out=gpu(4, 5, 128).transpose(0, 1)), 'output'),
    (attend, dict(out=gpu(5 * 4 * 128 + 8)[1:2561].view(5, 4, 128)), 'output'),
    (attend, dict(out=gpu(5, 4, 128, dtype=torch.float16)), 'share'),
    (attend, dict(lengths=gpu(2, dtype=F32)), 'int32'),
]


@pytest.mark.parametrize('run,change,message', REFUSED)
def test_refusals(calls, run, change, message):
    run()
    assert len(calls) == 1
    with pytest.raises(ValueError, match=message):
        run(**change)
    assert len(calls) == 1


def test_layouts_that_need_a_copy(calls):
    """Rows off 16 bytes, heads a stride of 4 apart and channels apart are copied first; other
    strides, and pages of one tensor with both, go to the library as they are."""
    off = gpu(5 * 4 * 128 + 8)[1:2561].view(5, 4, 128)
    wide = gpu(4, 5, 260).transpose(0, 1)[..., :128]
    for q in (off, wide, gpu(5, 4, 256)[..., ::2]):
        norm(q=q)
        name, args = calls.pop()
        assert args[0] % 16 == 0 and args[0] != q.data_ptr() and args[1:4] == (512, 128, 4)
    q = gpu(5, 4, 256)[..., 128:]
    both = gpu(6, 2, 2, 16, 128)
    attend(q=q, gate=gpu(4, 5, 128).transpose(0, 1), k_pages=both[:, 0], v_pages=both[:, 1])
    name, args = calls.pop()
    assert name == 'lm_paged_attention' and args[:4] == (q.data_ptr(), 1024, 256, 4)
    assert args[7] == 2 * 2 * 16 * 128


def rows_call(entry, **change):
    """The C call of an entry point with placeholder pointers, refused before any use."""
    at = 4096
    a = dict(q=at, q_token=512, q_head=128, q_heads=4, q_w=None, q_out=at, k=at, k_token=256,
             k_head=128, k_heads=2, k_w=None, k_out=at, v=at, positions=at, freq=at, pairs=32,
             tokens=5, dim=128, dtype=0, k_pages=at, v_pages=at, pages=6, page_stride=4096,
             page=16, starts=at, lengths=at, table=at, table_stride=3, table_pages=3, sequences=2,
             max_new=5, gate=None, gate_token=0, out=at, ws=at, ws_bytes=1 << 40)
    a.update(change)
    g = a.get
    batch = [g(n) for n in ('k_pages', 'v_pages', 'pages', 'page_stride', 'k_heads', 'page', 'dim',
                            'starts', 'lengths', 'table', 'table_stride', 'table_pages',
                            'sequences')]
    lib = _lib.lib()
    if entry == 'norm':
        rc = lib.lm_qk_norm_rope(*[g(n) for n in (
            'q', 'q_token', 'q_head', 'q_heads', 'q_w', 'q_out', 'k', 'k_token', 'k_head',
            'k_heads', 'k_w', 'k_out', 'positions', 'freq', 'pairs', 'tokens', 'dim')], 1e-6,
            g('dtype'), None)
    elif entry == 'append':
        rc = lib.lm_paged_append(*[g(n) for n in (
            'k', 'k_token', 'k_head', 'k_w', 'v', 'k_token', 'k_head', 'q', 'q_token', 'q_head',
            'q_heads', 'q_w', 'q_out')], *batch, g('freq'), g('pairs'), g('tokens'), 1e-6,
            g('dtype'), None)
    else:
        rc = lib.lm_paged_attention(*[g(n) for n in ('q', 'q_token', 'q_head', 'q_heads')], *batch,
                                    g('tokens'), g('max_new'), 0.1, g('gate'), g('gate_token'),
                                    128, g('out'), g('ws'), g('ws_bytes'), g('dtype'), None)
    return rc, lib.lm_last_error().decode()


ALL, PAGED = ('norm', 'append', 'attend'), ('append', 'attend')
C_REFUSED = [
    (ALL, dict(dtype=2), 'FP16/BF16'), (ALL, dict(dim=96), 'heads of'), (ALL, dict(q=4104), 'aligned'),
    (ALL, dict(q_token=516), 'aligned'), (ALL, dict(q_head=-128), 'aligned'),
    (ALL, dict(tokens=-1), 'token count'), (ALL, dict(tokens=1 << 31), 'token count'),
    (ALL, dict(q_heads=-2), 'heads'),
    (('norm', 'append'), dict(pairs=12), 'multiple of 16'),
    (('norm', 'append'), dict(pairs=72), 'multiple of 16'),
    (('norm', 'append'), dict(freq=None), 'null'), (('norm', 'append'), dict(k=None), 'aligned'),
    (('norm', 'append'), dict(k_w=4100), 'aligned'), (('norm', 'append'), dict(q_out=None), 'aligned'),
    (('norm',), dict(k_out=4104), 'aligned'), (('norm',), dict(positions=None), 'null'),
    (('append',), dict(v=None), 'aligned'),
    (PAGED, dict(page=24), 'page size'), (PAGED, dict(page=8), 'page size'),
    (PAGED, dict(page=2048), 'page size'), (PAGED, dict(pages=0), 'pages'),
    (PAGED, dict(page_stride=4088), 'pages'), (PAGED, dict(page_stride=4100), 'pages'),
    (PAGED, dict(k_heads=0), 'heads'), (PAGED, dict(starts=None), 'null'),
    (PAGED, dict(table=None), 'null'), (PAGED, dict(table_pages=0), 'page table'),
    (PAGED, dict(table_pages=1 << 27), 'page table'), (PAGED, dict(table_stride=-1), 'page table'),
    (PAGED, dict(sequences=-1), 'sequences'), (PAGED, dict(sequences=1 << 20), 'sequences'),
    (PAGED, dict(k_pages=None), ''), (PAGED, dict(v_pages=4104), 'aligned'),
    (('attend',), dict(q_heads=5), 'multiple'), (('attend',), dict(q_heads=0), 'multiple'),
    (('attend',), dict(max_new=-1), 'new tokens'), (('attend',), dict(out=None), 'null'),
    (('attend',), dict(out=4104), 'aligned'), (('attend',), dict(gate=4104), 'aligned'),
    (('attend',), dict(gate=4096, gate_token=4), 'aligned'),
]


@pytest.mark.parametrize('entry,change,message',
                         [(e, c, m) for es, c, m in C_REFUSED for e in es])
def test_c_refusals(entry, change, message):
    rc, error = rows_call(entry, **change)
    assert rc == _lib.LM_EINVAL and message in error


@pytest.mark.parametrize('entry', ALL)
def test_c_calls_without_work(entry):
    """No tokens, and no sequences: nothing is launched and no pointer is used."""
    assert rows_call(entry, tokens=0, q=None, k=None)[0] == _lib.LM_OK
    if entry != 'norm':
        assert rows_call(entry, sequences=0, q=None, k=None, starts=None)[0] == _lib.LM_OK


def test_c_sizes_of_a_launch():
    """More rows than a launch has threads for, and a scale that is none."""
    for entry in ALL:
        rc, error = rows_call(entry, tokens=1 << 24)
        assert rc == _lib.LM_EINVAL and 'token count' in error
    rc, error = rows_call('attend', k_heads=1024, q_heads=1024, q_token=1 << 17, page_stride=1 << 21,
                          sequences=65536)
    assert rc == _lib.LM_EINVAL and 'too many rows' in error
    rc, error = rows_call('attend', k_heads=1024, q_heads=1024, q_token=1 << 17, page_stride=1 << 21,
                          tokens=1 << 20, sequences=1 << 13, max_new=1 << 10)
    assert rc == _lib.LM_EINVAL and 'too many rows' in error


@pytest.mark.parametrize('scale', [float('nan'), float('inf')])
def test_c_scale_is_finite(scale, monkeypatch):
    def launch(device, name, *args):
        assert getattr(_lib.lib(), name)(*args, None) == _lib.LM_EINVAL
        raise ValueError(_lib.lib().lm_last_error().decode())
    monkeypatch.setattr(_lib, 'launch', launch)
    with pytest.raises(ValueError, match='finite'):
        attend(scale=scale)


@pytest.mark.parametrize('tokens,heads', [(1, 4), (1, 1), (5, 1), (2, 4)])
def test_layouts_of_few_rows(calls, tokens, heads):
    """A row pitch that the library does not take is copied for one token and one head too, where
    torch calls the rows contiguous whatever their strides are."""
    pitched = gpu(tokens, heads * 128 + 4)[:, :heads * 128].view(tokens, heads, 128)
    wide = gpu(tokens, heads, 132)[..., :128]
    odd = gpu(heads * 128).as_strided((1, heads, 128), (3, 128, 1))
    for q in (pitched, wide, odd)[:3 if tokens == 1 else 2]:
        n, h = q.shape[:2]
        norm(q=q, k=gpu(n, 2, 128), positions=gpu(n, dtype=I64))
        args = calls.pop()[1]
        assert args[0] % 16 == 0 and args[1] % 8 == 0 and args[2] % 8 == 0
        assert args[1] >= 0 and args[3] == h
        append(q=q, k=gpu(n, 2, 132)[..., :128], v=gpu(n, 2, 128))
        args = calls.pop()[1]
        assert all(args[i] % 8 == 0 for i in (1, 2, 5, 6, 8, 9))
        attend(q=q.expand(n, 4, 128), gate=wide.expand(n, 4, 128))
        args = calls.pop()[1]
        assert all(args[i] % 8 == 0 for i in (1, 2, 21, 22)) and args[0] % 16 == 0


def test_pages_whose_single_dimensions_have_other_strides(calls):
    """One key-value head, one page: their strides are stepped over by nothing."""
    one = gpu(6, 16, 1, 128).transpose(1, 2)  # [pages, page, heads, D] with a single head
    assert one.stride()[1] == 128 and one.is_contiguous()
    for k, v in ((one, one), (one, gpu(6, 1, 16, 128))):
        append(k_pages=k, v_pages=v, k=gpu(5, 1, 128), v=gpu(5, 1, 128))
        attend(k_pages=k, v_pages=v)
        for _, args in (calls.pop(0), calls.pop(0)):
            assert (6, 16 * 128, 1, 16, 128) in (args[15:20], args[6:11])
    first, last = gpu(6, 2, 2, 16, 128)[:1, 0], gpu(3, 2, 16, 128)[2:]
    attend(k_pages=first, v_pages=last)
    assert calls.pop()[1][6:11] == (1, 2 * 16 * 128, 2, 16, 128)
    for k, v in ((gpu(6, 1, 16, 128), gpu(6, 2, 1, 16, 128)[:, 0]),  # pages apart by another pitch
                 (gpu(6, 1, 32, 128)[:, :, ::2], gpu(6, 1, 32, 128)[:, :, ::2])):
        with pytest.raises(ValueError, match='pages|contiguous'):
            attend(k_pages=k, v_pages=v)


def test_a_cache_without_heads_is_refused(calls):
    with pytest.raises(ValueError, match='heads'):
        attend(k_pages=gpu(6, 0, 16, 128), v_pages=gpu(6, 0, 16, 128))
    assert not calls


@pytest.mark.parametrize('entry', PAGED)
@pytest.mark.parametrize('page,table_pages', [(16, (1 << 27) - 1), (64, (1 << 25) - 1), (1024, (1 << 21) - 1),
                                              (16, 1 << 60), (1024, 1 << 54)])
def test_c_tables_that_end_at_32_bits(entry, page, table_pages):
    """Kernels look up to 1024 positions past the one they are at, in 32 bits: a table that ends
    closer to 2^31 is refused, and so is one whose positions wrap around in 64 bits."""
    rc, error = rows_call(entry, page=page, table_pages=table_pages, page_stride=2 * page * 128)
    assert rc == _lib.LM_EINVAL and 'page table' in error
    rc, error = rows_call(entry, page=page, table_pages=(1 << 31) // page - 4096 // page, tokens=0,
                          page_stride=2 * page * 128)
    assert rc == _lib.LM_OK


@pytest.mark.parametrize('scale', [2.4e38, -3e38])
def test_c_scale_whose_exponent_is_finite(scale, monkeypatch):
    """The kernels work in powers of two: scale * log2(e) has to be a number too."""
    test_c_scale_is_finite(scale, monkeypatch)
