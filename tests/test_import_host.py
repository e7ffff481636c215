"""The package imports on builds of PyTorch that have no CUDA."""

import subprocess
import sys
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent


def test_import_without_the_cuda_bindings():
    """As in a CPU-only build: torch._C has no _cuda_* names that torch itself does not stub."""
    code = (
        "import torch\n"
        "for name in [n for n in dir(torch._C) if n.startswith('_cuda')]:\n"
        "    delattr(torch._C, name)\n"
        "import probe_b200\n"
        "x = torch.zeros(2, 32, dtype=torch.bfloat16)\n"
        "try:\n"
        "    probe_b200.mx_quantize(x)\n"
        "except RuntimeError as e:\n"
        "    assert 'CUDA' in str(e)\n"
        "else:\n"
        "    raise AssertionError('a CPU tensor was taken')\n"
    )
    run = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr
