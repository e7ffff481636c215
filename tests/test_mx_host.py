"""Microscaled tensors: the oracle's formats and the host-side checks (CPU only)."""

import ctypes

import numpy as np
import pytest
import torch

from oracle import mx_oracle as mo
from probe_b200 import _lib, mx


def test_oracle_grids():
    assert list(mo.E2M1) == [0, 0.5, 1, 1.5, 2, 3, 4, 6]
    assert mo.E4M3[-1] == 448 and len(mo.E4M3) == 127 and mo.E4M3[1] == 2.0 ** -9


def test_oracle_e4m3_rounding_is_torchs():
    v = torch.linspace(-440, 440, 40001)
    want = v.to(torch.float8_e4m3fn).double().numpy()
    got = np.copysign(mo.E4M3[mo.nearest(v.double().numpy(), mo.E4M3)], v.double().numpy())
    np.testing.assert_array_equal(got, want)


def test_oracle_ties_and_saturation():
    v = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.9, -0.25])
    np.testing.assert_array_equal(mo.E2M1[mo.nearest(v, mo.E2M1)], [0, 1, 1, 2, 2, 4, 4, 6, 0])


def test_scale_layout_is_one_byte_a_block():
    byte = np.arange(130 * 5).reshape(130, 5) % 251 + 1
    flat = mo.scale_layout(byte)
    assert flat.size == 2 * 2 * 512 and np.count_nonzero(flat) == 130 * 5
    assert flat[16 * 3 + 4 * 1 + 2] == byte[35, 2] and flat[3 * 512 + 16 * 1] == byte[129, 4]


@pytest.mark.parametrize("fmt,code", [("mxfp4", 0), ("nvfp4", 1), ("mxfp8", 2)])
@pytest.mark.parametrize("m,k", [(1, 1), (128, 128), (129, 4100)])
def test_sizes_agree_with_the_library(lib, fmt, code, m, k):
    pitch, scales = mx._sizes(m, k, fmt)
    assert lib.lora_mx_codes_size(m, k, code) == m * pitch
    assert lib.lora_mx_scales_size(m, k, code) == scales


def test_library_refuses_bad_arguments(lib):
    p = ctypes.c_void_p(256)
    q = lambda **kw: lib.lora_mx_quantize(*[{**dict(x=p, ldx=64, c=p, s=p, M=4, K=64, f=0, g=1.0, d=1, st=None),  # noqa: E731
                                             **kw}[n] for n in ("x", "ldx", "c", "s", "M", "K", "f", "g", "d", "st")])
    assert q(f=3) == _lib.LORA_ERR_DTYPE and q(d=2) == _lib.LORA_ERR_DTYPE
    assert q(ldx=63) == _lib.LORA_ERR_SHAPE and q(M=-1) == _lib.LORA_ERR_SHAPE
    assert q(g=2.0) == _lib.LORA_ERR_ARG and q(f=1, g=0.0) == _lib.LORA_ERR_ARG
    assert q(x=None) == _lib.LORA_ERR_ARG and q(c=ctypes.c_void_p(8)) == _lib.LORA_ERR_ALIGN
    assert q(M=0) == _lib.LORA_OK


def test_cpu_tensors_raise():
    with pytest.raises(RuntimeError, match="CUDA"):
        mx.mx_quantize(torch.zeros(2, 32, dtype=torch.bfloat16))


def test_global_scale_of_a_zero_tensor_is_usable():
    assert mx.nvfp4_global_scale(0.0) > 2.0 ** -64


@pytest.mark.parametrize("m,n,k,r", [(32760, 5120, 5120, 224), (256, 4096, 4096, 16), (4097, 11008, 4096, 20)])
def test_backward_workspace_has_no_copies_of_rows_read_in_place(lib, m, n, k, r):
    size = lambda flags: lib.lora_mx_backward_workspace_size(m, n, k, r, flags)  # noqa: E731
    dy, b = (-(-m * n * 2 // 256) * 256), (-(-r * n * 2 // 256) * 256)
    for dx in (0, _lib.LORA_MX_NEED_DX):
        bf16 = dx | _lib.LORA_MX_ONLY_BF16
        assert size(bf16) - size(bf16 | _lib.LORA_MX_DY_ALIGNED) == dy
        wide = r > 144 and m >= 24576  # such an adapter's g comes from B transposed
        assert size(bf16) - size(bf16 | _lib.LORA_MX_B_ALIGNED) == (0 if wide else b)
        assert size(dx) >= size(bf16)


def test_backward_workspace_keeps_the_copy_of_odd_rows(lib):
    """N no multiple of 8 is copied whatever the alignment of its first row."""
    size = lambda flags: lib.lora_mx_backward_workspace_size(512, 4097, 256, 16, flags)  # noqa: E731
    assert size(_lib.LORA_MX_DY_ALIGNED) == size(0)
