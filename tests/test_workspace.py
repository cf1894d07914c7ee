"""CPU checks of the pooled workspaces: an address that a captured launch may hold stays a zeroed buffer."""
import gc
import weakref

import pytest
import torch

import scope_b200
from scope_b200 import _lib


@pytest.fixture
def pool(monkeypatch):
    """A pool of CPU buffers for one device and stream."""
    monkeypatch.setattr(_lib, "stream_ptr", lambda device: 7)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "synchronize", lambda device=None: None)
    p = _lib._WorkspacePool()
    monkeypatch.setattr(_lib, "workspaces", p)
    return p


CPU = torch.device("cpu", 0)


def test_an_outgrown_workspace_stays(pool):
    first = pool.get(1 << 16, CPU)
    at, alive = first.data_ptr(), weakref.ref(first.untyped_storage())
    larger = pool.get(64 << 20, CPU)
    assert larger.numel() >= 64 << 20 and larger.data_ptr() != at
    assert pool.get(1 << 16, CPU) is larger
    del first
    gc.collect()
    assert alive() is not None
    assert any(b.data_ptr() == at for _, b in pool._outgrown)


def fake_status(monkeypatch, rc, what):
    class Fake:
        @staticmethod
        def ws_status_read(stream, out):
            out._obj.value = what
            return rc

    class Stream:
        cuda_stream = 0

    class Device:
        def __init__(self, d): pass
        def __enter__(self): pass
        def __exit__(self, *a): pass

    monkeypatch.setattr(scope_b200, "lib", lambda: Fake)
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda d=None: Stream)


def test_a_bad_index_leaves_workspaces_alone(pool, monkeypatch):
    buf = pool.get(1 << 16, CPU)
    buf[5] = 3   # a launch in flight
    fake_status(monkeypatch, _lib.WS_ERR_DEVICE, _lib.WS_STATUS_BAD_INDEX)
    assert scope_b200.status_take("cuda:0") == _lib.WS_ERR_DEVICE
    assert pool.get(1 << 16, CPU) is buf and buf[5] == 3


def test_a_timeout_zeroes_workspaces_where_they_lie(pool, monkeypatch):
    old = pool.get(1 << 16, CPU)
    buf = pool.get(64 << 20, CPU)
    old[0], buf[9] = 1, 2
    fake_status(monkeypatch, _lib.WS_ERR_DEVICE, _lib.WS_STATUS_TIMEOUT | _lib.WS_STATUS_BAD_INDEX)
    assert scope_b200.status_take("cuda:0") == _lib.WS_ERR_DEVICE
    assert pool.get(1 << 16, CPU) is buf and not buf.any() and not old.any()


def test_a_workspace_first_asked_for_in_a_capture_is_made_outside_of_it(pool, monkeypatch):
    made = []

    class Binding:
        @staticmethod
        def zeros_outside_capture(nbytes, index):
            made.append((nbytes, index))
            return torch.zeros(nbytes, dtype=torch.uint8)

    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    monkeypatch.setattr(_lib, "binding", lambda: Binding)
    buf = pool.get(1 << 16, CPU)
    assert made == [(pool.MIN_BYTES, 0)] and pool.get(1 << 16, CPU) is buf and len(made) == 1
