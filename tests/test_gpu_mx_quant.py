"""Microscaled quantisation: every code, scale byte and value against the float64 oracle."""

import numpy as np
import pytest
import torch

from oracle import mx_oracle as mo
from probe_b200 import _lib, mx

pytestmark = pytest.mark.gpu
DEV = "cuda"
FMTS = ("mxfp4", "nvfp4", "mxfp8")


def draw(m, k, dtype, seed=0):
    """Values over many binades, with runs of zeros, exact ties and both signs."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, k, generator=g) * torch.exp2(torch.randint(-12, 6, (m, 1), generator=g).float())
    x[torch.rand(m, k, generator=g) < 0.1] = 0.0
    x[:, : min(k, 16)] = torch.randint(-12, 13, (m, min(k, 16)), generator=g) / 4.0  # ties of E2M1
    x[m // 2] = 0.0
    return x.to(dtype)


def magnitudes(q):
    """Codes without the sign, one a value."""
    c = q.codes.cpu().numpy()
    if q.fmt == "mxfp8":
        return c & 0x7F
    return np.stack([c & 7, (c >> 4) & 7], axis=2).reshape(c.shape[0], -1)


def check(x, fmt, g=1.0):
    q = mx.mx_quantize(x.to(DEV), fmt, global_scale=g)
    codes, byte, val = mo.quantize(x.double().numpy(), fmt, g)
    np.testing.assert_array_equal(magnitudes(q), codes)
    np.testing.assert_array_equal(q.scales.cpu().numpy(), mo.scale_layout(byte))
    for dtype in (torch.bfloat16, torch.float16):
        # the value is formed in float32 and rounded once more: exact products first
        want = torch.from_numpy(val).float().to(dtype)
        got = mx.mx_dequantize(q, dtype)
        assert torch.equal(got.cpu().nan_to_num(7.0), want.nan_to_num(7.0))
        assert torch.equal(mx.mx_dequantize(q, dtype, transpose=True).nan_to_num(7.0), got.t().nan_to_num(7.0))
    return q


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m,k", [(1, 1), (1, 32), (3, 31), (2, 130), (127, 64), (128, 128), (129, 257), (300, 96)])
def test_codes_scales_and_values(fmt, dtype, m, k):
    check(draw(m, k, dtype), fmt, 2.0 ** -9 if fmt == "nvfp4" else 1.0)


@pytest.mark.parametrize("g", [1.0, 0.0123, 3.7e-5, 2.0 ** -60, 2.0 ** 60])
def test_nvfp4_global_scales(g):
    """Block scales that saturate (g small) or vanish (g large)."""
    check(draw(40, 200, torch.bfloat16, seed=3), "nvfp4", float(np.float32(g)))


@pytest.mark.parametrize("fmt", FMTS)
def test_extreme_magnitudes(fmt):
    """The type's largest and smallest values, and subnormal ones."""
    for dtype in (torch.bfloat16, torch.float16):
        fi = torch.finfo(dtype)
        x = torch.zeros(4, 64, dtype=dtype)
        x[0] = fi.max
        x[1, ::2] = fi.tiny
        x[2] = fi.smallest_normal / 4
        x[3, 5], x[3, 40] = -fi.max, fi.tiny
        q = mx.mx_quantize(x.to(DEV), fmt)
        codes, byte, val = mo.quantize(x.double().numpy(), fmt)
        np.testing.assert_array_equal(magnitudes(q), codes)
        np.testing.assert_array_equal(q.scales.cpu().numpy(), mo.scale_layout(byte))


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_non_finite_blocks(fmt, value):
    x = draw(5, 96, torch.bfloat16, seed=1)
    x[1, 40] = value
    x[4, 0] = value
    q = check(x, fmt, 2.0 ** -7 if fmt == "nvfp4" else 1.0)
    v = mx.mx_dequantize(q)
    size = mo.BLOCK[fmt]
    first = 40 // size * size
    assert v[1, first:first + size].isnan().all() and v[4, :size].isnan().all()
    assert int(v.isnan().sum()) == 2 * size


@pytest.mark.parametrize("fmt", FMTS)
def test_strided_and_unaligned_input(fmt):
    x = draw(70, 203, torch.bfloat16, seed=2).to(DEV)
    g = 2.0 ** -8 if fmt == "nvfp4" else 1.0
    for view in (x[:, 3:], x[::2, :64], x.t(), x[5:6, 1:2], x[:, 8:136]):
        a, b = mx.mx_quantize(view, fmt, g), mx.mx_quantize(view.contiguous(), fmt, g)
        assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)


@pytest.mark.parametrize("fmt", FMTS)
def test_leading_dimensions_and_empty(fmt):
    x = draw(24, 64, torch.float16).to(DEV)
    a, b = mx.mx_quantize(x.view(2, 3, 4, 64), fmt), mx.mx_quantize(x, fmt)
    assert a.shape == (24, 64) and torch.equal(a.codes, b.codes)
    e = mx.mx_quantize(x[:0], fmt)
    assert e.shape == (0, 64) and mx.mx_dequantize(e).shape == (0, 64)


def test_other_stream():
    x = draw(513, 1024, torch.bfloat16).to(DEV)
    want = mx.mx_quantize(x, "mxfp4")
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = mx.mx_dequantize(mx.mx_quantize(x, "mxfp4"))
    s.synchronize()
    assert torch.equal(got, mx.mx_dequantize(want))


def test_refusals():
    x = torch.zeros(4, 64, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError, match="unknown format"):
        mx.mx_quantize(x, "fp4")
    with pytest.raises(RuntimeError, match="CUDA"):
        mx.mx_quantize(x.cpu(), "mxfp4")
    with pytest.raises(TypeError):
        mx.mx_quantize(x.float(), "mxfp4")
    for g in (0.0, -1.0, float("nan"), float("inf"), 1e-30):
        with pytest.raises(_lib.LoraValueError):
            mx.mx_quantize(x, "nvfp4", global_scale=g)
    with pytest.raises(_lib.LoraValueError):
        mx.mx_quantize(x, "mxfp4", global_scale=2.0)
    q = mx.mx_quantize(x, "mxfp4")
    with pytest.raises(TypeError):
        mx.mx_dequantize(q, torch.float32)
    with pytest.raises(ValueError):
        mx.MXTensor(q.codes, q.scales, (4, 128), "mxfp4")
    with pytest.raises(ValueError):
        mx.MXTensor(q.codes[:, ::2], q.scales, (4, 32), "mxfp4")
    with pytest.raises(TypeError):
        mx.MXTensor(q.codes.int(), q.scales, (4, 64), "mxfp4")
