"""Which kernels may share an SM with the shrink of a wide adapter.

A CTA waits for tensor memory that another holds.  A thread-block cluster waits for its
CTAs, so a CTA that holds tensor memory may wait for one that waits for tensor memory:
two clustered kernels of two streams could wait for one another for good.  The SM's shared
memory rules it out: a kernel that takes all 512 columns leaves none of it for another.
"""

import json

import pytest
import torch
from torch.profiler import ProfilerActivity, profile

from probe_b200 import mx
from tests.test_gpu_mx_linear import G, case

pytestmark = pytest.mark.gpu

SM_BYTES = 228 * 1024  # shared memory of an SM; a CTA's own and 1 KB more are taken from it
SMALLEST = 2 * 128 * 128  # two stages of 128 rows of 64 16-bit columns: no kernel with tensor memory has less


@pytest.mark.parametrize("m,k,r", [(40, 512, 130), (64, 512, 224), (200, 512, 170), (200, 512, 224), (300, 512, 250)])
@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_nothing_joins_a_cta_with_all_of_tensor_memory(tmp_path, m, k, r, fmt):
    x, wq, bi, a, b, _ = case(m, 136, k, r, torch.bfloat16, fmt)
    run = lambda: mx.mx_lora_linear(x, wq, bi, a, b, 1.0, x_global_scale=G[fmt][0])  # noqa: E731
    run()
    torch.cuda.synchronize()
    with profile(activities=[ProfilerActivity.CUDA]) as p:
        run()
        torch.cuda.synchronize()
    p.export_chrome_trace(str(tmp_path / "trace.json"))
    events = json.loads((tmp_path / "trace.json").read_text())["traceEvents"]
    taken = [e["args"]["shared memory"] for e in events if e.get("cat") == "kernel" and "mx_shrink" in e["name"]]
    assert taken and min(taken) + 1024 + SMALLEST + 1024 > SM_BYTES
