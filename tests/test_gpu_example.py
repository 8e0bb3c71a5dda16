"""The example of a whole training step: all operators with the optimizer."""

import importlib.util
from pathlib import Path

import pytest

from gpu_util import announce, needs_gpu

pytestmark = [pytest.mark.gpu, needs_gpu]


def test_distill_adapters_learns_and_repeats():
    announce("example distill_adapters")
    path = Path(__file__).resolve().parents[1] / "examples" / "distill_adapters.py"
    spec = importlib.util.spec_from_file_location("distill_adapters", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    losses = example.train(steps=40)
    assert losses[-1] < 0.8 * losses[0], losses
    assert example.train(steps=5) == losses[:5]   # every kernel on the way sums in a fixed order
