"""MXLoRALinear under autograd: second derivatives, scale 0."""

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


@pytest.mark.parametrize("m", [3, 300])
@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_scale_zero_trains_as_it_serves(fmt, m):
    """The adapter is off: its gradients are zeros, y and dx are the base's."""
    mod = module(0.0, fmt)
    x = randn((m, 96), 1.0, torch.bfloat16, 4).requires_grad_()
    dy = randn((m, 64), 1.0, torch.bfloat16, 5)
    with torch.no_grad():
        served = mod(x)
    y = mod(x)
    assert torch.equal(y, served)
    y.backward(dy)
    assert not mod.lora_a.grad.any() and not mod.lora_b.grad.any()
    x8 = mx.mx_quantize(x.detach(), "mxfp8")
    off = torch.zeros_like(mod.lora_b)
    want, _, _ = mx.mx_lora_backward(dy, x8, torch.zeros(m, 32, dtype=dy.dtype, device=DEV), mod.lora_a.detach(), off,
                                     1.0, weight=mod.weight)
    assert torch.equal(x.grad, want)
