"""Gradients of wide adapters on both sides of the rows from which g has a GEMM of its own."""

import pytest
import torch

from probe_b200 import _lib, mx
from tests.test_gpu_mx_backward import case, check, formulas
from tests.test_gpu_mx_gradient_precision import pair_formulas

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,n,k,r", [(24575, 72, 96, 150), (24576, 72, 96, 150), (25001, 137, 64, 224), (24600, 64, 288, 256)])
def test_rows(m, n, k, r, dtype):
    dy, x8, z, a, b, w = case(m, n, k, r, dtype, seed=23)
    got = mx.mx_lora_backward(dy, x8, z, a, b, 1.3, weight=w)
    want = formulas(dy, x8, z, a, b, w, 1.3, 1.0, dtype)
    want.update(pair_formulas(dy, x8, z, a, b, 1.3, dtype))
    check(got, want)
    assert _lib.device_error(0) == 0
