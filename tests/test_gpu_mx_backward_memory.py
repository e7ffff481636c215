"""The backward pass takes no memory for copies that it does not make, and has room for those it does."""

import pytest
import torch

from probe_b200 import _lib, mx
from tests.test_gpu_mx_backward import case, check, formulas

pytestmark = pytest.mark.gpu


def test_a_training_step_holds_no_copy_of_dy():
    m, n, k, r = 16384, 4096, 512, 16
    dy, x8, z, a, b, _ = case(m, n, k, r, torch.bfloat16)
    s = torch.cuda.Stream()  # a workspace of its own
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    with torch.cuda.stream(s):
        out = mx.mx_lora_backward(dy, x8, z, a, b, 1.0)
    s.synchronize()
    held = torch.cuda.memory_allocated() - before - sum(t.numel() * 2 for t in out if t is not None)
    assert held < m * n * 2 / 4


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,n,k,r", [(200, 328, 256, 24), (4100, 136, 1288, 136), (300, 72, 9608, 20)])
def test_rows_of_every_alignment_have_their_room(m, n, k, r, dtype):
    """Aligned, then not, on a stream whose workspace is as small as the first call needs."""
    dy, x8, z, a, b, w = case(m, n, k, r, dtype, seed=19)
    wide = torch.zeros(m, n + 8, dtype=dtype, device="cuda")
    wide[:, 3:3 + n] = dy
    bt = torch.zeros(n, r + 5, dtype=dtype, device="cuda")
    bt[:, 1:1 + r] = b
    want = formulas(dy, x8, z, a, b, w, 1.0, 1.0, dtype)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        for d in (dy, wide[:, 3:3 + n]):
            for bb in (b, bt[:, 1:1 + r]):
                check(mx.mx_lora_backward(d, x8, z, a, bb, 1.0, weight=w), want)
    assert _lib.device_error(0) == 0
