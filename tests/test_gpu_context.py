"""The library leaves the driver context that its caller made current."""

import ctypes
import threading

import pytest
import torch

from probe_b200 import _lib

pytestmark = pytest.mark.gpu


def in_a_thread(fn):
    out = []
    t = threading.Thread(target=lambda: out.append(fn()))
    t.start()
    t.join()
    assert len(out) == 1, "the thread raised"
    return out[0]


def query():
    """An entry point that asks for the current device and launches nothing."""
    return _lib.load().lora_mx_backward_workspace_size(16, 64, 64, 4, 0)


def test_a_context_of_the_callers_stays_current():
    cuda = ctypes.CDLL("libcuda.so.1")
    torch.zeros(1, device="cuda")
    size = query()

    def run():
        dev, ctx, now = ctypes.c_int(), ctypes.c_void_p(), ctypes.c_void_p()
        assert cuda.cuDeviceGet(ctypes.byref(dev), torch.cuda.current_device()) == 0
        assert cuda.cuCtxCreate_v2(ctypes.byref(ctx), 0, dev) == 0
        try:
            assert query() == size
            assert cuda.cuCtxGetCurrent(ctypes.byref(now)) == 0
            return now.value == ctx.value
        finally:
            cuda.cuCtxDestroy_v2(ctx)

    assert in_a_thread(run)


def test_a_thread_without_a_context_gets_the_primary_one():
    cuda = ctypes.CDLL("libcuda.so.1")
    torch.zeros(1, device="cuda")
    primary = ctypes.c_void_p()
    assert cuda.cuCtxGetCurrent(ctypes.byref(primary)) == 0 and primary.value

    def run():
        now = ctypes.c_void_p()
        assert cuda.cuCtxGetCurrent(ctypes.byref(now)) == 0 and not now.value
        query()
        assert cuda.cuCtxGetCurrent(ctypes.byref(now)) == 0
        return now.value

    assert in_a_thread(run) == primary.value
