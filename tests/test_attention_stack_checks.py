"""CPU checks of MoEStack with attention layers: what a step refuses, that it refuses before it
queues anything, and how its two streams are ordered when a call fails.  Streams and layers only
record what is asked of them."""
import contextlib

import pytest
import torch

from localmoe35ba3b_amd.runtime.stack import MoEStack
from tests.test_attention_block_checks import H, batch, block, pages
from tests.test_attention_checks import gpu


class Stream:
    def __init__(self, name, log):
        self.name, self.log = name, log

    def wait_stream(self, other):
        self.log.append((self.name, 'waits for', other.name))

    def wait_event(self, event):
        self.log.append((self.name, 'waits for', event))


class Event:
    def record(self, stream):
        stream.log.append((stream.name, 'records', self))


@pytest.fixture
def step(monkeypatch):
    """make(attention) gives a stack of three layers of 64 rows at most, and the log of what it
    queues, in order."""
    log, at = [], ['caller']
    caller, side = Stream('caller', log), Stream('side', log)

    @contextlib.contextmanager
    def on(stream):
        before, at[0] = at[0], stream.name
        try:
            yield
        finally:
            at[0] = before

    monkeypatch.setattr(torch.cuda, 'stream', on)
    monkeypatch.setattr(torch.cuda, 'Event', Event)
    monkeypatch.setattr(torch.cuda, 'current_stream', lambda device=None: caller)

    def make(attention):
        st = MoEStack.__new__(MoEStack)
        st.L, st.H, st.max_tokens, st.device = 3, H, 64, torch.device('cpu')
        st.workspace, st._side, st._side_ws = None, side, None
        st._tiles_of = None
        st.layer_forward = lambda h, l, **kw: log.append((at[0], 'layer', l))
        st.attention = attention
        for l, b in attention.items():
            b.queue = lambda h, batch, l=l: log.append((at[0], 'attention', l))
            b.forward_ = b.queue
        return st, log

    return make


@pytest.mark.parametrize('fails_at', [0, 1, 2])
def test_overlapped_prefill_joins_its_streams_when_a_call_fails(step, fails_at):
    """A layer that fails with work of the second stream queued: the caller's stream waits for that
    work all the same, as it writes the caller's rows."""
    st, log = step({1: pages(block())})
    calls = []

    def fails(h, batch):
        if len(calls) == fails_at:
            raise MemoryError('no memory for a workspace')
        calls.append(1)
        log.append('attention')

    st.attention[1].forward_ = fails
    with pytest.raises(MemoryError, match='no memory'):
        st.prefill_(gpu(48, H), 16, batch=batch())
    assert ('side', 'layer', 0) in log
    assert log[-1] == ('caller', 'waits for', 'side')


def test_overlapped_prefill_joins_its_streams(step):
    st, log = step({1: pages(block())})
    st.prefill_(gpu(48, H), 16, batch=batch())
    assert log[0] == ('side', 'waits for', 'caller') and log[-1] == ('caller', 'waits for', 'side')
    assert sum(e[1:] == ('attention', 1) for e in log) == 3
    assert sum(e[1] == 'layer' for e in log) == 9


def run_forward(st, h, batch):
    st.forward(h, batch=batch)


def run_prefill(st, h, batch):
    st.prefill_(h, 16, batch=batch)


def run_prefill_alone(st, h, batch):
    st.prefill_(h, 16, overlap=False, batch=batch)


RUNS = pytest.mark.parametrize('run', [run_forward, run_prefill, run_prefill_alone])
I32, I64 = torch.int32, torch.int64


@RUNS
@pytest.mark.parametrize('change,message', [
    (dict(starts=gpu(2, dtype=I64)), 'int32'), (dict(lengths=gpu(1, dtype=I64)), 'int32'),
    (dict(table=gpu(1, 3, dtype=I64)), 'int32'), (dict(starts=gpu(3, dtype=I32)), 'match'),
    (dict(table=gpu(3, dtype=I32)), 'match'), (dict(max_new=-1), 'new tokens')])
def test_batches_are_refused_before_anything_is_queued(step, run, change, message):
    st, log = step({2: pages(block())})
    run(st, gpu(48, H), batch())
    assert len(log) > 3
    log.clear()
    with pytest.raises(ValueError, match=message):
        run(st, gpu(48, H), batch(**change))
    assert not log


@RUNS
def test_caches_are_refused_before_anything_is_queued(step, run):
    for late, kind, message in (
            (block(), RuntimeError, 'allocate'), (pages(block(), torch.float16), ValueError, 'share'),
            (pages(block(kv_heads=1)), ValueError, 'heads'),
            (pages(block(head_dim=128)), ValueError, 'heads')):
        st, log = step({0: pages(block()), 2: late})
        with pytest.raises(kind, match=message):
            run(st, gpu(48, H), batch())
        assert not log


def test_rows_are_refused_before_attention_writes_them(step):
    """As without attention, where the first layer refuses them."""
    st, log = step({0: pages(block())})
    for h, kind in ((gpu(65, H), MemoryError), (gpu(4, H, dtype=torch.float16), ValueError),
                    (gpu(4, 2 * H)[:, ::2], ValueError), (gpu(4, H + 128), ValueError),
                    (gpu(1, 4, H), ValueError)):
        with pytest.raises(kind):
            st.forward(h, batch=batch())
    st._tiles_of, st._bank_versions = (0, 0), lambda: (1, 0)
    for run in (run_forward, run_prefill, run_prefill_alone):
        with pytest.raises(RuntimeError, match='build_prefill_tiles'):
            run(st, gpu(48, H), batch())
    st._tiles_of = None
    st.E, st.I, st.K, st.H = 256, 512, 8, 2048
    st.attention = {0: pages(wide())}
    with pytest.raises(MemoryError, match='workspace'):
        st.forward(gpu(4, 2048), workspace=gpu(1024, dtype=torch.uint8), batch=batch())
    assert not log


def wide():
    """A block of the stack's own width."""
    b = block()
    b.qkv = {k: v[:, :1].expand(-1, 2048 if k == 'q' else 16) for k, v in b.qkv.items()}
    return b


def test_layers_that_do_not_run_need_no_batch(step):
    for run in (run_forward, run_prefill, run_prefill_alone):
        st, log = step({3: pages(block())})
        run(st, gpu(48, H), None)
        assert sum(e[1] == 'layer' for e in log) == (3 if run is run_forward else 9)
        log.clear()
    st, log = step({1: block()})
    st.forward(gpu(4, H), layers=1)
    assert log == [('caller', 'layer', 0)]


def test_step_in_order(step):
    st, log = step({0: pages(block()), 2: pages(block())})
    st.forward(gpu(4, H), batch=batch())
    assert [e[1:] for e in log] == [('attention', 0), ('layer', 0), ('layer', 1), ('attention', 2),
                                    ('layer', 2)]


def test_batches_are_read_by_name(step):
    """A program's own batch object serves as before."""
    import types
    st, log = step({0: pages(block())})
    st.forward(gpu(4, H), batch=types.SimpleNamespace(**batch()._asdict()))
    assert len(log) == 4
