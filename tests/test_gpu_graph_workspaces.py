"""CUDA graphs and the workspaces they were captured with."""

import pytest
import torch

from probe_b200 import kernels, mx
from tests.helpers import randn

pytestmark = pytest.mark.gpu
DEV = "cuda"


def operands(n, k, r, fmt="mxfp4"):
    w = mx.mx_quantize(randn((n, k), k ** -0.5, torch.bfloat16, 1), fmt, 2.0 ** -12 if fmt == "nvfp4" else 1.0)
    return w, randn((r, k), k ** -0.5, torch.bfloat16, 2), randn((n, r), 0.2, torch.bfloat16, 3)


def linear(m, k=1024, n=512):
    w, a, b = operands(n, k, 16)
    x = randn((m, k), 1.0, torch.bfloat16, 4)
    return lambda: [mx.mx_lora_linear(x, w, None, a, b, 2.0)]


def backward(m, k=512, n=512):
    w, a, b = operands(n, k, 16)
    dy, z = randn((m, n), 1.0, torch.bfloat16, 4), randn((m, 32), 1.0, torch.bfloat16, 5)
    x8 = mx.mx_quantize(randn((m, k), 1.0, torch.bfloat16, 6), "mxfp8")
    return lambda: list(mx.mx_lora_backward(dy, x8, z, a, b, 2.0, weight=w))


def shrink(m, k=4096):
    x, a = randn((m, k), 1.0, torch.bfloat16, 7), randn((32, k), k ** -0.5, torch.bfloat16, 8)
    return lambda: [kernels.shrink(x, a, 1.0, split_k=4)]


@pytest.mark.parametrize("make,small,large", [(linear, 16, 6000), (backward, 40, 5000), (shrink, 64, 9000)])
def test_a_larger_call_after_the_capture(make, small, large):
    """The workspace grows; the graph's own stays, and nothing else comes to lie there."""
    s = torch.cuda.Stream()
    few, many = make(small), make(large)
    with torch.cuda.stream(s):
        want = [t.clone() for t in few()]
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        got = few()
    with torch.cuda.stream(s):
        many()
        # tensors over whatever the growth gave back
        others = [torch.full((size,), 0xA5, dtype=torch.uint8, device=DEV)
                  for size in (1 << 12, 1 << 16, 1 << 18, 1 << 19, 1 << 20, 1 << 21, 1 << 22) for _ in range(16)]
    for _ in range(3):
        for t in got:
            t.zero_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want))
        assert all(bool((t == 0xA5).all()) for t in others)


@pytest.mark.parametrize("make,few", [(linear, 16), (linear, 700), (backward, 40), (shrink, 64)])
def test_captures_without_a_warm_call(make, few):
    """Two graphs captured on one stream that had no workspace yet, replayed in the other order, then eagerly."""
    first, second = make(few), make(few + 8)
    want = [[t.clone() for t in f()] for f in (first, second)]  # on another stream: the kernels are loaded
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    graphs, outs = [], []
    for f in (first, second):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(f())
        graphs.append(g)
    for i in (1, 0, 1, 1, 0):
        for t in outs[i]:
            t.zero_()
        graphs[i].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(outs[i], want[i]))
    with torch.cuda.stream(s):
        again = first()
    s.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(again, want[0]))
