"""The LoRA linear with 4-bit base operands against the float64 oracle."""

import numpy as np
import pytest
import torch

from oracle import mx_oracle as mo
from probe_b200 import _lib, mx
from tests.helpers import dtype_tag, np64, randn

pytestmark = pytest.mark.gpu
DEV = "cuda"
G = {"mxfp4": (1.0, 1.0), "nvfp4": (float(np.float32(9.1 / 2688)), float(np.float32(0.31 / 2688)))}


def case(m, n, k, r, dtype, fmt, bias=True, seed=0):
    x = randn((m, k), 2.0, dtype, seed)
    w = randn((n, k), k ** -0.5, dtype, seed + 1)
    a = randn((r, k), k ** -0.5, dtype, seed + 2) if r else None
    b = randn((n, r), max(r, 1) ** -0.5, dtype, seed + 3) if r else None
    return x, mx.mx_quantize(w, fmt, G[fmt][1]), (randn((n,), 1.0, dtype, seed + 4) if bias else None), a, b, w


def want(x, w, bias, a, b, scale, fmt, dtype):
    """Reference and elementwise bound; w: the 16-bit weight that was quantised."""
    gx, gw = G[fmt]
    k = x.shape[1]
    qx, qw = mo.quantize(np64(x), fmt, gx)[2], mo.quantize(np64(w), fmt, gw)[2]
    ref, mass = qx @ qw.T, np.abs(qx) @ np.abs(qw).T
    extra = 0.0
    if a is not None:
        z = scale * (np64(x) @ np64(a).T)
        zmass = abs(scale) * (np.abs(np64(x)) @ np.abs(np64(a)).T)
        ref = ref + z @ np64(b).T
        lora = np.abs(z) @ np.abs(np64(b)).T
        mass = mass + lora
        # z: a float32 sum, kept as a hi/lo pair (two 8- or 11-bit parts)
        pair = 2.0 ** -16 if dtype == torch.bfloat16 else 2.0 ** -21
        extra = pair * lora + (k / 16 + 8) * 2.0 ** -23 * (zmass @ np.abs(np64(b)).T)
    if bias is not None:
        ref, mass = ref + np64(bias), mass + np.abs(np64(bias))
    return ref, mo.product_bound(ref, mass, k, dtype_tag(dtype), extra)


def check(y, ref, bound):
    err = np.abs(np64(y) - ref)
    assert y.shape == ref.shape and np.isfinite(np64(y)).all()
    assert (err <= bound).all(), f"worst {np.max(err / bound):.2f} of the bound"


SIZES = [
    (1, 64, 32, 4, False), (1, 300, 1024, 16, True), (3, 257, 96, 1, True), (17, 128, 416, 33, False),
    (64, 1000, 2080, 16, True), (128, 256, 256, 64, False), (129, 513, 544, 20, True), (256, 512, 1024, 128, False),
    (257, 264, 288, 130, True), (600, 768, 1120, 224, True), (1025, 520, 512, 256, False), (70, 96, 64, 0, True),
    (300, 640, 768, 0, False), (2100, 2304, 320, 8, True),
    (2560, 2304, 320, 224, False), (2500, 2400, 288, 32, True),  # more tiles than CTA pairs, long and short tails
    # the same for outputs and lengths that end inside a tile, rows of every alignment
    (2000, 2313, 256, 16, True), (1300, 2050, 96, 20, True), (1500, 1976, 544, 130, False), (2100, 2304, 32, 4, True),
    (1411, 2311, 1000, 8, False), (19000, 136, 64, 6, True),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("m,n,k,r,bias", SIZES)
def test_against_oracle(m, n, k, r, bias, fmt, dtype):
    x, wq, bi, a, b, w = case(m, n, k, r, dtype, fmt, bias)
    y = mx.mx_lora_linear(x, wq, bi, a, b, 1.7, x_global_scale=G[fmt][0])
    check(y, *want(x, w, bi, a, b, 1.7, fmt, dtype))
    assert _lib.device_error(0) == 0


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_odd_k_pads_with_zeros(fmt):
    """K that is no multiple of 32: the padded columns count for nothing."""
    x, wq, bi, a, b, w = case(40, 72, 1000, 8, torch.bfloat16, fmt)
    check(mx.mx_lora_linear(x, wq, bi, a, b, 0.5, G[fmt][0]), *want(x, w, bi, a, b, 0.5, fmt, torch.bfloat16))
    x, wq, bi, a, b, w = case(300, 260, 333, 8, torch.bfloat16, fmt)
    check(mx.mx_lora_linear(x, wq, bi, a, b, 0.5, G[fmt][0]), *want(x, w, bi, a, b, 0.5, fmt, torch.bfloat16))


@pytest.mark.parametrize("m", [5, 300])
def test_strides_and_leading_dimensions(m):
    x, wq, bi, a, b, w = case(m, 200, 256, 24, torch.bfloat16, "mxfp4")
    base = mx.mx_lora_linear(x, wq, bi, a, b, 2.0)
    wide = torch.zeros(m, 300, dtype=x.dtype, device=DEV)
    wide[:, 7:263] = x
    at = torch.zeros(256, 30, dtype=x.dtype, device=DEV)
    at[:, 3:27] = a.t()
    bt = torch.zeros(200, 33, dtype=x.dtype, device=DEV)
    bt[:, 1:25] = b
    got = mx.mx_lora_linear(wide[:, 7:263], wq, bi, at[:, 3:27].t(), bt[:, 1:25], 2.0)
    assert torch.equal(got, base)
    assert torch.equal(mx.mx_lora_linear(x.view(1, m, 256), wq, bi, a, b, 2.0), base[None])


@pytest.mark.parametrize("m", [1, 64, 300])
def test_repeats_bitwise_and_on_another_stream(m):
    x, wq, bi, a, b, _ = case(m, 1024, 2048, 16, torch.bfloat16, "nvfp4")
    first = mx.mx_lora_linear(x, wq, bi, a, b, 2.0, G["nvfp4"][0])
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        other = mx.mx_lora_linear(x, wq, bi, a, b, 2.0, G["nvfp4"][0])
    s.synchronize()
    assert torch.equal(first, other)
    for _ in range(3):
        assert torch.equal(first, mx.mx_lora_linear(x, wq, bi, a, b, 2.0, G["nvfp4"][0]))


@pytest.mark.parametrize("m", [4, 200, 520])
def test_a_nan_stays_in_its_row(m):
    x, wq, bi, a, b, _ = case(m, 320, 512, 8, torch.bfloat16, "mxfp4")
    base = mx.mx_lora_linear(x, wq, bi, a, b, 2.0)
    x[2, 100] = float("nan")
    y = mx.mx_lora_linear(x, wq, bi, a, b, 2.0)
    assert y[2].isnan().all()
    keep = torch.arange(m, device=DEV) != 2
    assert torch.equal(y[keep], base[keep])


def test_tiny_tensor_scales():
    """Tensor scales whose product needs more than one power-of-two step (fp16 z stays finite)."""
    m, n, k, r = 300, 256, 512, 16
    x, w = randn((m, k), 2e-3, torch.float16, 1), randn((n, k), 1e-3, torch.float16, 2)
    a, b = randn((r, k), k ** -0.5, torch.float16, 3), randn((n, r), 0.02, torch.float16, 4)
    gx, gw = float(np.float32(9e-3 / 2688)), float(np.float32(5e-3 / 2688))
    for mm in (m, 7):
        y = mx.mx_lora_linear(x[:mm], mx.mx_quantize(w, "nvfp4", gw), None, a, b, 1.0, gx)
        qx, qw = mo.quantize(np64(x[:mm]), "nvfp4", gx)[2], mo.quantize(np64(w), "nvfp4", gw)[2]
        z = np64(x[:mm]) @ np64(a).T
        ref = qx @ qw.T + z @ np64(b).T
        lora = np.abs(z) @ np.abs(np64(b)).T
        zm = (np.abs(np64(x[:mm])) @ np.abs(np64(a)).T) @ np.abs(np64(b)).T
        check(y, ref, mo.product_bound(ref, np.abs(qx) @ np.abs(qw).T + lora, k, "fp16",
                                       2.0 ** -21 * lora + (k / 16 + 8) * 2.0 ** -23 * zm))


@pytest.mark.parametrize("m", [16, 400])
def test_graph_capture(m):
    x, wq, bi, a, b, _ = case(m, 512, 1024, 16, torch.bfloat16, "mxfp4")
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        want_y = mx.mx_lora_linear(x, wq, bi, a, b, 2.0)
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        y = mx.mx_lora_linear(x, wq, bi, a, b, 2.0)
    y.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want_y)


def test_empty():
    x, wq, bi, a, b, _ = case(2, 64, 64, 8, torch.bfloat16, "mxfp4")
    assert mx.mx_lora_linear(x[:0], wq, bi, a, b).shape == (0, 64)


def test_refusals():
    x, wq, bi, a, b, w = case(4, 64, 96, 8, torch.bfloat16, "mxfp4")
    with pytest.raises(ValueError, match="4-bit"):
        mx.mx_lora_linear(x, mx.mx_quantize(w, "mxfp8"), bi, a, b)
    with pytest.raises(ValueError, match="disagree"):
        mx.mx_lora_linear(x[:, :64], wq, bi, a, b)
    with pytest.raises(ValueError):
        mx.mx_lora_linear(x, wq, bi, a[:, :64], b)
    with pytest.raises(ValueError):
        mx.mx_lora_linear(x, wq, bi[:10], a, b)
    with pytest.raises(TypeError):
        mx.mx_lora_linear(x, wq, bi, a.half(), b)
    with pytest.raises(TypeError):
        mx.mx_lora_linear(x.float(), wq, bi, a, b)
    with pytest.raises(RuntimeError, match="CUDA"):
        mx.mx_lora_linear(x.cpu(), wq, bi, a, b)
    with pytest.raises(ValueError, match="256"):
        big = torch.zeros(300, 96, dtype=x.dtype, device=DEV)
        mx.mx_lora_linear(x, wq, None, big, torch.zeros(64, 300, dtype=x.dtype, device=DEV))
    with pytest.raises(_lib.LoraValueError):
        mx.mx_lora_linear(x, wq, bi, a, b, 1.0, x_global_scale=2.0)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("m", [1, 16, 17, 33, 64, 65, 300, 2100])
def test_another_call_leaves_nothing_behind(m, fmt):
    """Quantised rows beyond the tokens hold what an earlier call left there: here NaN."""
    n, k, r = 2304, 320, 8
    x, wq, bias, a, b, w = case(m, n, k, r, torch.bfloat16, fmt, seed=31)
    spoilt = torch.full(((m + 127) // 128 * 128, k), float("inf"), dtype=torch.bfloat16, device=DEV)
    assert torch.isnan(mx.mx_lora_linear(spoilt, wq, bias, a, b, 1.7, x_global_scale=G[fmt][0])).all()
    y = mx.mx_lora_linear(x, wq, bias, a, b, 1.7, x_global_scale=G[fmt][0])
    check(y, *want(x, w, bias, a, b, 1.7, fmt, torch.bfloat16))


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("m,k,r", [(1, 13824, 64), (23, 13824, 16), (60, 6912, 200), (8343, 1184, 64), (4119, 2048, 40)])
def test_long_rows_of_few_tokens(m, k, r, fmt):
    """Many more tiles along K than stages, in blocks of few rows among others."""
    n = 136
    x, wq, bias, a, b, w = case(m, n, k, r, torch.bfloat16, fmt, seed=41)
    for _ in range(3):
        y = mx.mx_lora_linear(x, wq, bias, a, b, 0.8, x_global_scale=G[fmt][0])
    check(y, *want(x, w, bias, a, b, 0.8, fmt, torch.bfloat16))
