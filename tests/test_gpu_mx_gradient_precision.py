"""What the adapter's gradients keep of g = s dy B and of z: both halves of the pair at
every rank, and, for fp16 activations, values of g on both sides of fp16's range."""

import numpy as np
import pytest
import torch

from oracle import mx_oracle as mo
from probe_b200 import mx
from tests.helpers import dtype_tag, np64, randn
from tests.test_gpu_mx_backward import GW, case, check, formulas, values

pytestmark = pytest.mark.gpu
DEV = "cuda"


def pair_formulas(dy, x8, z, a, b, scale, dtype):
    """(reference, elementwise bound) of da and db whose g and z are pairs at any rank: an
    error of one rounding of a rounding in each term, the float32 sums, one rounding."""
    d, xv, bv = np64(dy), values(x8), np64(b)
    m, n = d.shape
    r, r16 = b.shape[1], z.shape[1] // 2
    tag = dtype_tag(dtype)
    pair = (2.0 ** -8 if tag == "bf16" else 2.0 ** -11) ** 2
    zv = np64(z[:, :r]) + np64(z[:, r16:r16 + r])
    g = scale * d @ bv
    gacc = (n / 16 + 8) * 2.0 ** -23 * abs(scale) * (np.abs(d) @ np.abs(bv))
    da, dam = g.T @ xv, np.abs(g).T @ np.abs(xv)
    db, dbm = d.T @ zv, np.abs(d).T @ np.abs(zv)
    return {"da": (da, mo.product_bound(da, dam, m, tag, pair * dam + gacc.T @ np.abs(xv))),
            "db": (db, mo.product_bound(db, dbm, m, tag, pair * dbm))}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,n,k,r", [(65, 520, 288, 65), (130, 264, 544, 96), (700, 200, 160, 128), (1, 64, 96, 130),
                                     (300, 96, 1000, 224), (513, 264, 520, 256), (4100, 264, 288, 200),
                                     (4099, 130, 96, 144)])
def test_both_halves_above_rank_64(m, n, k, r, dtype):
    dy, x8, z, a, b, _ = case(m, n, k, r, dtype, seed=17)
    check(mx.mx_lora_backward(dy, x8, z, a, b, 1.7), pair_formulas(dy, x8, z, a, b, 1.7, dtype))


RANGE = [(6, 40, 64, 4), (300, 256, 256, 16), (200, 264, 136, 40), (300, 72, 9608, 20), (300, 96, 1000, 224),
         (4097, 136, 1288, 136)]


def ranged(m, n, k, r, fmt, dy_exp, b_exp, x_exp, a_exp):
    """A case whose dy, B, X and A lie about the given powers of two."""
    dy, _, z, a, b, w = case(m, n, k, r, torch.float16, fmt, seed=29)
    x8 = mx.mx_quantize(randn((m, k), 2.0 ** x_exp, torch.float16, 30), "mxfp8")
    return (dy * 2.0 ** dy_exp, x8, z, randn((r, k), 2.0 ** a_exp, torch.float16, 31),
            randn((n, r), 2.0 ** b_exp, torch.float16, 32), w)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("m,n,k,r", RANGE)
def test_fp16_g_below_its_range(m, n, k, r, fmt):
    """B just off zero, as LoRA training starts: g about 2^-22, dA well inside fp16."""
    dy, x8, z, a, b, w = ranged(m, n, k, r, fmt, -10, -14, 9, -4)
    check(mx.mx_lora_backward(dy, x8, z, a, b, 1.0, weight=w), formulas(dy, x8, z, a, b, w, 1.0, 1.0, torch.float16))


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("m,n,k,r", RANGE)
def test_fp16_g_above_its_range(m, n, k, r, fmt):
    """g beyond 65504 with gradients that fp16 holds."""
    dy, x8, z, a, b, w = ranged(m, n, k, r, fmt, 6, 9, -14, -14)
    g = np64(dy) @ np64(b)
    assert np.abs(g).max() > 65504
    check(mx.mx_lora_backward(dy, x8, z, a, b, 1.0, weight=w), formulas(dy, x8, z, a, b, w, 1.0, 1.0, torch.float16))
