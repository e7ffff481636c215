"""The 4-bit LoRA linear above rank 128 with rows of any length and alignment."""

import pytest
import torch

from probe_b200 import mx
from tests.helpers import np64
from tests.test_gpu_mx_backward import check as check_gradients
from tests.test_gpu_mx_backward import formulas
from tests.test_gpu_mx_linear import G, case, check, want

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("m,n,k,r", [(1, 64, 35, 129), (5, 72, 333, 130), (300, 264, 1001, 224), (2500, 2056, 70, 256)])
def test_k_of_any_size(m, n, k, r, fmt, dtype):
    x, wq, bi, a, b, w = case(m, n, k, r, dtype, fmt)
    y = mx.mx_lora_linear(x, wq, bi, a, b, 1.7, x_global_scale=G[fmt][0])
    check(y, *want(x, w, bi, a, b, 1.7, fmt, dtype))


@pytest.mark.parametrize("k", [256, 260])
def test_rows_of_any_layout(k):
    m, n, r = 140, 96, 136
    x, wq, bi, a, b, w = case(m, n, k, r, torch.bfloat16, "mxfp4")
    ref = want(x, w, bi, a, b, 2.0, "mxfp4", torch.bfloat16)
    base = mx.mx_lora_linear(x, wq, bi, a, b, 2.0)
    check(base, *ref)
    wide = torch.zeros(m, k + 11, dtype=x.dtype, device=DEV)
    wide[:, 3:3 + k] = x
    pitched = torch.zeros(m, 264, dtype=x.dtype, device=DEV)
    pitched[:, :k] = x
    at = torch.zeros(k, r + 5, dtype=x.dtype, device=DEV)
    at[:, 1:1 + r] = a.t()
    for xv in (x, wide[:, 3:3 + k], pitched[:, :k]):
        for av in (a, at[:, 1:1 + r].t()):
            assert torch.equal(mx.mx_lora_linear(xv, wq, bi, av, b, 2.0), base)


def test_training_forward():
    m, n, k, r = 210, 120, 333, 144
    x, wq, bi, a, b, w = case(m, n, k, r, torch.bfloat16, "nvfp4")
    y, x8, z, zs = mx.mx_lora_forward(x, wq, bi, a, b, 0.5, G["nvfp4"][0])
    check(y, *want(x, w, bi, a, b, 0.5, "nvfp4", torch.bfloat16))
    exact = 0.5 * np64(x) @ np64(a).T
    got = zs * (np64(z[:, :r]) + np64(z[:, r:2 * r]))
    mass = 0.5 * abs(np64(x)) @ abs(np64(a)).T
    assert (abs(got - exact) <= 2.0 ** -16 * abs(exact) + (k / 16 + 8) * 2.0 ** -23 * mass).all()
    dy = torch.randn(m, n, device=DEV).to(torch.bfloat16)
    check_gradients(mx.mx_lora_backward(dy, x8, z, a, b, 0.5, weight=wq, z_scale=zs),
                    formulas(dy, x8, z, a, b, wq, 0.5, zs, torch.bfloat16))
