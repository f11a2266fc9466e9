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
