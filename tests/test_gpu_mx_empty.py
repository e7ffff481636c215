"""Gradients of the 4-bit LoRA linear where a dimension is empty."""

import ctypes

import pytest
import torch

from probe_b200 import _lib, mx
from tests.helpers import randn

pytestmark = pytest.mark.gpu
DEV = "cuda"


def nan(*shape):
    return torch.full(shape, float("nan"), dtype=torch.bfloat16, device=DEV)


def backward(m, n, k, r, da, db, dx):
    """The C entry on outputs that hold NaN."""
    p = lambda t: ctypes.c_void_p(t.data_ptr()) if t.numel() else ctypes.c_void_p(256)  # noqa: E731
    z = randn((m, 2 * ((r + 15) // 16 * 16)), 1.0, torch.bfloat16, 1)
    dy, a, b = (randn(s, 1.0, torch.bfloat16, i) for i, s in enumerate(((m, n), (r, k), (n, r))))
    x8 = mx.mx_quantize(randn((m, k), 1.0, torch.bfloat16, 7), "mxfp8")
    w = mx.mx_quantize(randn((n, k), 1.0, torch.bfloat16, 8), "mxfp4")
    lib = _lib.load()
    ws = torch.zeros(max(lib.lora_mx_backward_workspace_size(m, n, k, r, 1), 256), dtype=torch.uint8, device=DEV)
    return lib.lora_mx_backward(p(dy), n, p(x8.codes), p(x8.scales), p(z), 1.0, p(a), k, p(b), r, p(w.codes),
                                p(w.scales), 1.0, _lib.LORA_MXFP4, p(dx), k, p(da), k, p(db), r, m, n, k, r, 1.0,
                                _lib.LORA_BF16, p(ws), ws.numel(), torch.cuda.current_stream().cuda_stream)


@pytest.mark.parametrize("m", [1, 40, 600])
def test_no_outputs(m):
    """N = 0: dy is empty, so dA and dx are sums over nothing."""
    k, r = 96, 8
    da, db, dx = nan(r, k), nan(0, r), nan(m, k)
    assert backward(m, 0, k, r, da, db, dx) == _lib.LORA_OK
    assert not da.any() and not dx.any()


def test_no_outputs_through_the_wrapper():
    m, k, r = 12, 64, 4
    a, b = randn((r, k), 1.0), nan(0, r)
    w = mx.mx_quantize(randn((1, k), 1.0)[:0], "nvfp4", 2.0 ** -9)
    x8 = mx.mx_quantize(randn((m, k), 1.0), "mxfp8")
    junk = [nan(m, k) for _ in range(4)]  # what the allocator hands out next held NaN
    del junk
    dx, da, db = mx.mx_lora_backward(nan(m, 0), x8, randn((m, 32), 1.0), a, b, 1.0, weight=w)
    assert dx.shape == (m, k) and not dx.any() and da.shape == (r, k) and not da.any() and db.shape == (0, r)


def test_no_inputs_is_refused_as_in_the_forward_pass():
    """K = 0: dB = dy^T z does not depend on K and would be left unwritten."""
    da, db, dx = nan(8, 0), nan(64, 8), nan(40, 0)
    assert backward(40, 64, 0, 8, da, db, dx) == _lib.LORA_ERR_UNSUPPORTED
