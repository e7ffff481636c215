"""An MXLoRALinear saved and loaded again gives the same outputs and gradients."""

import io

import pytest
import torch
from torch import nn

from probe_b200 import mx
from tests.helpers import randn

pytestmark = pytest.mark.gpu
DEV = "cuda"


def module(fmt, std, seed, n=96, k=160, r=8, x_amax=32.0):
    base = nn.Linear(k, n, device=DEV, dtype=torch.bfloat16)
    with torch.no_grad():
        base.weight.copy_(randn((n, k), std, torch.bfloat16, seed))
    return mx.MXLoRALinear(base, randn((r, k), 0.1, torch.bfloat16, seed + 1), randn((n, r), 0.3, torch.bfloat16, seed + 2),
                           1.5, fmt, x_amax)


def outputs(mod, x, dy):
    x = x.detach().requires_grad_()
    y = mod(x)
    return (y.detach(), *torch.autograd.grad(y, (x, mod.lora_a, mod.lora_b), dy))


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_round_trip_into_a_module_of_another_base(fmt):
    """The tensor-wide scales of nvfp4 (of W, and the input's calibration) travel with the codes."""
    src, dst = module(fmt, 0.7, 1, x_amax=9.0), module(fmt, 0.02, 11)
    x, dy = randn((33, 160), 2.0, torch.bfloat16, 5), randn((33, 96), 1.0, torch.bfloat16, 6)
    want = outputs(src, x, dy)
    file = io.BytesIO()
    torch.save(src.state_dict(), file)
    file.seek(0)
    result = dst.load_state_dict(torch.load(file, weights_only=True))
    assert not result.missing_keys and not result.unexpected_keys
    for got, ref in zip(outputs(dst, x, dy), want):
        assert torch.equal(got, ref)


def test_a_module_inside_another():
    src, dst = (nn.Sequential(module("nvfp4", std, 3), nn.ReLU(), module("nvfp4", std, 7, n=32, k=96)) for std in (0.4, 0.01))
    x = randn((5, 160), 1.0, torch.bfloat16, 5)
    dst.load_state_dict(src.state_dict())
    with torch.no_grad():
        assert torch.equal(dst(x), src(x))


def test_another_format_is_refused():
    """Codes of the two 4-bit formats have one shape; at K = 32 their scales do too."""
    for a, b in (("mxfp4", "nvfp4"), ("nvfp4", "mxfp4")):
        with pytest.raises(RuntimeError, match="mxfp4"):
            module(a, 0.1, 1, k=32).load_state_dict(module(b, 0.1, 1, k=32).state_dict())


def test_states_without_tensor_scales():
    """mxfp4 has none to restore; nvfp4 codes mean nothing without theirs."""
    for fmt in ("mxfp4", "nvfp4"):
        src, dst = module(fmt, 0.7, 1), module(fmt, 0.02, 11)
        state = {k: v for k, v in src.state_dict().items() if not k.endswith("_extra_state")}
        if fmt == "nvfp4":
            with pytest.raises(RuntimeError, match="_extra_state"):
                dst.load_state_dict(state)
            continue
        dst.load_state_dict(state)
        x = randn((4, 160), 1.0, torch.bfloat16, 5)
        with torch.no_grad():
            assert torch.equal(dst(x), src(x))
