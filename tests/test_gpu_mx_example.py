"""The example that trains and serves through the 4-bit LoRA linear runs and learns."""

import importlib.util
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_example(fmt):
    path = Path(__file__).resolve().parent.parent / "examples" / "mx_lora.py"
    spec = importlib.util.spec_from_file_location("mx_lora_example", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    got = mod.main(["--hidden", "512", "--ffn", "1376", "--tokens", "700", "--steps", "20", "--fmt", fmt])
    assert got["last"] < 0.9 * got["first"]
    assert got["weight_bytes"] < 0.3 * got["dense_bytes"] and got["kept_bytes"] < 0.53 * got["input_bytes"]
