"""Who hears of a router product whose wait gave up: every workspace on its device, once each, and
together with the workspace's own failures.  The library and the device are stand-ins here; the test
that expires a real wait is marked ``gpu``."""
import contextlib
import ctypes
import types

import pytest
import torch

from gc_moe_b200 import _native, operator
from gc_moe_b200.buffer import GCSymmBuffer


class FakeLibrary:
    """Status words of two devices; ``plans`` maps a plan's handle to the code it answers."""

    def __init__(self):
        self.current, self.stream_of, self.plans, self.failed, self.asked = 0, {}, {}, {0: False, 1: False}, []

    def gcmoe_producer_status(self, stream, words):
        self.asked.append((self.current, stream.value))
        failed, self.failed[self.current] = self.failed[self.current], False
        self.message = f'device wait gave up: kernel 5 on {self.current}'
        return _native.ERR_DEVICE if failed else 0

    def gcmoe_status_read(self, handle, stream, words):
        self.message = f'device wait gave up: kernel 1 of {handle}'
        return self.plans[handle]

    def gcmoe_last_error(self):
        return self.message.encode()


@pytest.fixture
def fake(monkeypatch):
    lib = FakeLibrary()

    @contextlib.contextmanager
    def device(d):
        before, lib.current = lib.current, torch.device(d).index
        yield
        lib.current = before

    def current_stream(d=None):
        return types.SimpleNamespace(cuda_stream=0x10 + (lib.current if d is None else torch.device(d).index))

    monkeypatch.setattr(_native, 'library', lambda: lib)
    monkeypatch.setattr(torch.cuda, 'device', device)
    monkeypatch.setattr(torch.cuda, 'current_stream', current_stream)
    return lib


def _workspace(index):
    w = GCSymmBuffer.__new__(GCSymmBuffer)
    w.buffer = types.SimpleNamespace(device=torch.device('cuda', index))
    w._plans, w._retired_scratch = {}, []
    w._producer_failures_seen = operator.producer_failures(w.buffer.device)
    return w


def test_every_workspace_of_the_device_hears_once(fake):
    first, second, elsewhere = _workspace(0), _workspace(0), _workspace(1)
    fake.failed[0] = True
    with pytest.raises(RuntimeError, match='kernel 5 on 0'):
        first.raise_on_device_error()
    first.raise_on_device_error()
    elsewhere.raise_on_device_error()
    with pytest.raises(RuntimeError, match='kernel 5 on 0'):
        second.raise_on_device_error()
    second.raise_on_device_error()
    _workspace(0).raise_on_device_error()                 # made after the failure had been read
    fake.failed[0] = True
    for w in (second, first):
        with pytest.raises(RuntimeError, match='kernel 5 on 0'):
            w.raise_on_device_error()


def test_the_workspaces_device_is_asked(fake):
    w = _workspace(1)
    fake.failed[1] = True
    with pytest.raises(RuntimeError, match='kernel 5 on 1'):
        w.raise_on_device_error()                         # the current device is 0
    assert fake.asked == [(1, 0x11)] and fake.current == 0


def test_a_producers_failure_does_not_hide_the_workspaces_own(fake):
    w = _workspace(0)
    w._plans = {'a': types.SimpleNamespace(handle='a'), 'b': types.SimpleNamespace(handle='b')}
    fake.plans = {'a': 0, 'b': _native.ERR_DEVICE}
    fake.failed[0] = True
    with pytest.raises(RuntimeError) as error:
        w.raise_on_device_error()
    assert 'kernel 5 on 0' in str(error.value) and 'kernel 1 of b' in str(error.value)


@pytest.mark.gpu
def test_an_expired_wait_reaches_every_workspace(single_rank_group):
    import gc_moe_b200 as G
    lib = _native.library()
    buffers = [G.get_symm_buffer_for_gc_moe(single_rank_group, 8, 256, 2, 1024, 512) for _ in range(2)]
    try:
        for b in buffers:
            b.raise_on_device_error()
        words = (ctypes.c_uint32 * _native.STATUS_WORDS)()
        other = torch.cuda.Stream()                       # the product of the second workspace runs elsewhere
        _native.raise_for(lib.gcmoe_debug_expire_producer_wait(200, ctypes.c_void_p(other.cuda_stream)))
        other.synchronize()
        for b in buffers:
            with pytest.raises(RuntimeError, match='gave up: code 1 kernel 5 site 99'):
                b.raise_on_device_error()
            b.raise_on_device_error()
        stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
        assert lib.gcmoe_producer_status(stream, words) == 0 and words[0] == 0
    finally:
        for b in buffers:
            b.destroy()
