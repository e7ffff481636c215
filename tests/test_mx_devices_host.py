"""Which GPU a microscaled call runs on (CPU only: tensors are stand-ins that are never read)."""

import contextlib
import types

import pytest
import torch

from probe_b200 import mx


def on(index, *shape, dtype=torch.bfloat16):
    """What the argument checks see of a CUDA tensor."""
    return types.SimpleNamespace(shape=torch.Size(shape), dtype=dtype, is_cuda=True, get_device=lambda: index,
                                 device=torch.device("cuda", index), is_contiguous=lambda: True,
                                 requires_grad=False)


def held(index, m, k, fmt="mxfp4"):
    return types.SimpleNamespace(codes=on(index, m, k // 2, dtype=torch.uint8), shape=(m, k), fmt=fmt,
                                 _code=mx._FORMATS[fmt], global_scale=1.0)


@pytest.fixture
def current(monkeypatch):
    """The current device, as torch.cuda.device sets it."""
    state = types.SimpleNamespace(index=0, entered=[])

    @contextlib.contextmanager
    def device(d):
        before, state.index = state.index, torch.device(d).index
        state.entered.append(state.index)
        try:
            yield
        finally:
            state.index = before

    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(mx, "_current_device", lambda: state.index)
    return state


N, K, R, M = 64, 96, 8, 5
LINEAR = dict(x=(M, K), bias=(N,), a=(R, K), b=(N, R))


@pytest.mark.parametrize("other", ["weight", "bias", "a", "b"])
def test_linear_refuses_operands_of_another_device(current, other):
    t = {k: on(int(k == other), *v) for k, v in LINEAR.items()}
    with pytest.raises(ValueError, match="different devices"):
        mx.mx_lora_linear(t["x"], held(int(other == "weight"), N, K), t["bias"], t["a"], t["b"])


@pytest.mark.parametrize("other", ["x8", "z", "a", "b", "weight"])
def test_backward_refuses_operands_of_another_device(current, other):
    at = lambda name: int(name == other)  # noqa: E731
    with pytest.raises(ValueError, match="different devices"):
        mx.mx_lora_backward(on(0, M, N), held(at("x8"), M, K, "mxfp8"), on(at("z"), M, 32), on(at("a"), R, K),
                            on(at("b"), N, R), weight=held(at("weight"), N, K))


def test_calls_run_on_the_device_of_their_tensors(current):
    """The kernels launch on the current device: it has to be the tensors'."""
    with pytest.raises(ValueError, match="disagree on K"):
        mx.mx_lora_linear(on(1, M, K + 32), held(1, N, K), None, None, None)
    with pytest.raises(ValueError, match="mxfp8"):
        mx.mx_lora_backward(on(1, M, N), held(1, M, K), on(1, M, 32), on(1, R, K), on(1, N, R))
    with pytest.raises(TypeError):
        mx.mx_quantize(on(1, M, K, dtype=torch.float32))
    with pytest.raises(TypeError):
        mx.mx_dequantize(held(1, M, K), dtype=torch.float32)
    assert current.entered == [1, 1, 1, 1] and current.index == 0
    with pytest.raises(TypeError):
        mx.mx_quantize(on(0, M, K, dtype=torch.float32))
    assert len(current.entered) == 4
