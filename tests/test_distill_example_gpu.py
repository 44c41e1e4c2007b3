"""The distillation example: sampling, loss and optimiser steps together."""
import importlib.util
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu


def test_distill_policy_example(cuda):
    path = Path(__file__).resolve().parents[1] / "examples" / "distill_policy.py"
    spec = importlib.util.spec_from_file_location("distill_policy", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    losses, before, after = mod.main(["--steps", "150", "--batch", "1024"])
    assert losses[-1] < losses[0] and after > before
