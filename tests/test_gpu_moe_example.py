"""examples/moe_distill_step.py runs, and training lowers its loss."""
import importlib.util
import math
import os

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_training_by_distillation_lowers_the_loss(bcjr_mod):
    spec = importlib.util.spec_from_file_location("moe_distill_step", os.path.join(ROOT, "examples", "moe_distill_step.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    losses = m.main(steps=12, tokens=200, verbose=False)
    assert all(math.isfinite(x) for x in losses)
    assert min(losses[6:]) < losses[0]
