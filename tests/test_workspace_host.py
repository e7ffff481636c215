"""Who holds a workspace, and for how long (CPU only: the stream and its capture are stand-ins)."""

import gc
import types
import weakref

import pytest
import torch

from probe_b200 import _lib

CPU = torch.device("cpu")


@pytest.fixture
def gpu(monkeypatch):
    """One stream, capturing when told to."""
    state = types.SimpleNamespace(capturing=False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: types.SimpleNamespace(cuda_stream=7))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: state.capturing)
    return state


def test_a_captured_buffer_outlives_its_replacement(gpu):
    """A graph replays with the address it was captured with."""
    ws = _lib._Workspace()
    ws.get(5000, CPU, "linear")
    gpu.capturing = True
    taken = weakref.ref(ws.get(5000, CPU, "linear"))
    gpu.capturing = False
    assert ws.get(4_000_000, CPU, "linear").numel() >= 4_000_000
    gc.collect()
    assert taken() is not None


def test_what_no_capture_took_is_given_back(gpu):
    ws = _lib._Workspace()
    first = weakref.ref(ws.get(5000, CPU, "linear"))
    gpu.capturing = True
    ws.get(100, CPU, "backward")
    gpu.capturing = False
    ws.get(4_000_000, CPU, "linear")
    gc.collect()
    assert first() is None


def test_a_buffer_serves_every_smaller_call(gpu):
    ws = _lib._Workspace()
    buf = ws.get(9000, CPU, "linear")
    assert ws.get(9000, CPU, "linear") is buf and ws.get(1, CPU, "linear") is buf
    assert ws.get(1, CPU, "linear", stream=7) is buf and ws.get(1, CPU, "linear", stream=8) is not buf
    assert ws.get(1, CPU, "backward") is not buf and not buf.any()


def test_a_buffer_of_a_capture_serves_that_call_alone(gpu):
    """Its zeros are written when the graph is replayed: not before another call, and not for another graph."""
    ws = _lib._Workspace()
    gpu.capturing = True
    first, second = ws.get(5000, CPU, "linear"), ws.get(5000, CPU, "linear")
    gpu.capturing = False
    eager = ws.get(5000, CPU, "linear")
    assert len({t.data_ptr() for t in (first, second, eager)}) == 3
    gpu.capturing = True
    assert ws.get(5000, CPU, "linear") is eager  # warmed now
    assert ws.get(9000, CPU, "linear") is not eager
    gpu.capturing = False
    assert ws.get(5000, CPU, "linear") is eager


def test_growth_doubles_small_buffers_and_not_large_ones(gpu):
    ws, mb = _lib._Workspace(), 1 << 20
    assert ws.get(5 * mb, CPU, "a").numel() == 5 * mb
    assert ws.get(6 * mb, CPU, "a").numel() == 10 * mb
    ws.get(300 * mb, CPU, "b")
    assert ws.get(301 * mb, CPU, "b").numel() == 364 * mb
    assert ws.get(500 * mb, CPU, "b").numel() == 500 * mb
