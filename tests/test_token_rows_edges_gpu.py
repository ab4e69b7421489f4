"""Token scoring and distillation at single edges of what the entry points
accept, against the float64 oracle (oracle/token_ops.py)."""
import numpy as np
import pytest

from oracle import token_ops as ops
from tests.helpers import Dev
from tests.test_token_rows_gpu import Rows, all_three, distill, teacher_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return Dev()


# a cluster, a CTA and a warp per row
SHAPES = [(4, 20001), (4, 3001), (452, 600)]


@pytest.mark.parametrize("rows,vocab", SHAPES)
@pytest.mark.parametrize("shift", [-1000, -200, -80, 0, 80, 200, 1000])
@pytest.mark.parametrize("tau", [1.0, 2.0])
def test_nothing_outside_the_slots_far_from_zero(dev, rows, vocab, shift, tau):
    """Every token outside the slots at -inf and logits away from 0, with a
    target in a slot and one outside.  The slots hold all of the teacher's
    mass but a millionth, which is below the bounds."""
    rng = np.random.default_rng(51)
    _, ids, teacher = teacher_of(rng, rows, vocab, 16)
    teacher = np.log(rng.dirichlet(np.ones(16), rows)).astype(np.float32)
    z = np.full((rows, vocab), -np.inf)
    np.put_along_axis(z, ids.astype(np.int64), shift + rng.standard_normal((rows, 16)), 1)
    targets = ids[:, 3].copy()
    targets[1::4] = [int(np.setdiff1d(np.arange(vocab), ids[i])[0]) for i in range(1, rows, 4)]
    targets[2::4] = ops.NO_TOKEN
    for tail in (False, True):
        one, two, both = all_three(dev, Rows(dev, z), ids, teacher, None, tail=tail, targets=targets, ce=0.5, tau=tau)
        masked = np.isneginf(z)
        masked[np.arange(rows), np.where(targets < vocab, targets, 0)] = False
        for got in (two, both):
            assert not got["grad"][masked].any()
