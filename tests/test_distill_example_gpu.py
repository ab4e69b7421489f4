"""The distillation example (examples/distill.py): scoring, the distillation
step and the policy step together, through the C ABI."""
import importlib.util
import os

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_the_student_follows_its_teacher():
    spec = importlib.util.spec_from_file_location("distill_example", os.path.join(ROOT, "examples", "distill.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    got = example.run(steps=40, policy_steps=5, report=lambda line: None)
    kl = np.array([k for _, k in got["history"]])
    assert np.isfinite(got["history"]).all() and np.isfinite(got["policy"]).all()
    # the divergence falls by more than half, and steps up its gradient raise
    # the given tokens' log probability
    assert kl[-1] < 0.5 * kl[0], kl
    assert got["policy"][-1] > got["policy"][0], got["policy"]
