"""The example that trains, quantises and decodes a gated-recurrence stack, run small."""

from __future__ import annotations

import importlib.util
import math
from pathlib import Path

import pytest

PATH = Path(__file__).resolve().parents[1] / "examples" / "train_quantize_decode.py"


def _run(*argv):
    spec = importlib.util.spec_from_file_location("train_quantize_decode", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module.main(list(argv))


def test_cpu():
    result = _run("--device", "cpu", "--width", "32", "--depth", "1", "--length", "32", "--batch", "2", "--steps", "3",
                  "--group-size", "32")
    assert all(math.isfinite(v) for v in result.values())
    # the same float32 formulas, by sequence or by token: only the order of the recurrence's products differs
    assert result["decoding"] < 1e-5


@pytest.mark.gpu
def test_gpu():
    result = _run("--device", "cuda", "--width", "128", "--length", "96", "--steps", "30")
    assert all(math.isfinite(v) for v in result.values())
    # bfloat16 activations between layers, rounded after sums in another order: some units of 2^-8, over two layers
    assert result["decoding"] < 8 * 2.0 ** -8
    assert result["last_loss"] < result["first_loss"]
