"""MXLoRALinear under autograd: second derivatives."""

import pytest
import torch
from torch import nn

from probe_b200 import mx
from tests.helpers import randn

pytestmark = pytest.mark.gpu
DEV = "cuda"


def module(scale, fmt="mxfp4", n=64, k=96, r=8):
    base = nn.Linear(k, n, device=DEV, dtype=torch.bfloat16)
    with torch.no_grad():
        base.weight.copy_(randn((n, k), 0.1, torch.bfloat16, 1))
    return mx.MXLoRALinear(base, randn((r, k), 0.1, torch.bfloat16, 2), randn((n, r), 0.3, torch.bfloat16, 3), scale, fmt)


def test_second_derivatives_raise():
    """A gradient penalty must not lose its term without a word."""
    mod = module(1.0)
    x = randn((20, 96), 1.0, torch.bfloat16, 4).requires_grad_()
    y = mod(x)
    (dx,) = torch.autograd.grad(y.float().square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        (y.float().sum() + dx.float().square().sum()).backward()
