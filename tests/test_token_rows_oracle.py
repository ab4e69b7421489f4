"""The float64 oracle of token scoring and distillation (oracle/token_ops.py)
against its own definition: gradients against central differences, known
values by hand.  CPU only.

Difference tolerance: central differences of step 1e-5 in float64 are off by
step^2 |f'''| / 6 ~ 1e-10 and by rounding 1e-16 |f| / step ~ 1e-10 for
losses of order 10."""
import numpy as np
import pytest

from oracle import token_ops as ops

STEP = 1e-5


def differences(f, z):
    g = np.zeros_like(z)
    for i in range(z.shape[0]):
        for j in range(z.shape[1]):
            if np.isneginf(z[i, j]):
                continue
            a, b = z.copy(), z.copy()
            a[i, j] += STEP
            b[i, j] -= STEP
            g[i, j] = (f(a)[i] - f(b)[i]) / (2 * STEP)
    return g


@pytest.mark.parametrize("temperature", [0.5, 1.0, 3.0])
def test_scoring_gradient_against_differences(temperature):
    rng = np.random.default_rng(3)
    z = rng.standard_normal((4, 13)) * 2
    z[1, [0, 5]] = -np.inf
    t = np.array([3, 2, ops.NO_TOKEN, 12], np.uint32)
    gl, ge = rng.standard_normal(4), rng.standard_normal(4)
    want = differences(lambda x: gl * ops.logprob(x, t, temperature)
                       + ge * ops.entropy(x, temperature), z)
    np.testing.assert_allclose(ops.logprob_gradient(z, t, gl, ge, temperature), want, atol=2e-9)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("temperature,ce", [(1.0, 0.0), (2.0, 0.3)])
def test_distillation_gradient_against_differences(tail, temperature, ce):
    rng = np.random.default_rng(4)
    z = rng.standard_normal((5, 11)) * 2
    z[2, 9] = -np.inf
    ids = np.array([[1, 4, 7], [0, 10, 3], [5, 6, 2], [8, ops.NO_TOKEN, 1],
                    [ops.NO_TOKEN] * 3], np.uint32)
    u = np.log(np.array([[.5, .2, .1], [.3, .3, .3], [.9, .05, .01], [.4, .4, .2], [.3, .3, .3]]))
    t = np.array([4, 2, 0, ops.NO_TOKEN, 6], np.uint32)
    args = dict(temperature=temperature, tail=tail, targets=t, kd=0.7, ce=ce)
    want = differences(lambda x: ops.distill(x, ids, u, **args)[0], z)
    np.testing.assert_allclose(ops.distill_gradient(z, ids, u, **args), want, atol=2e-9)


def test_known_values():
    z = np.log(np.array([[.5, .25, .25], [.5, .25, .25], [1, 1, 1]]))
    np.testing.assert_allclose(ops.logprob(z, [0, 2, ops.NO_TOKEN]), [np.log(.5), np.log(.25), 0])
    np.testing.assert_allclose(ops.entropy(z), [1.5 * np.log(2), 1.5 * np.log(2), np.log(3)])
    assert ops.top(z, 3).tolist() == [[0, 1, 2], [0, 1, 2], [0, 1, 2]]
    # the teacher is the student: no divergence, and no gradient
    ids = np.array([[0, 1], [0, 2], [1, 2]], np.uint32)
    u = np.take_along_axis(z, ids.astype(int), 1)
    u = u - np.log(np.exp(z).sum(-1, keepdims=True))
    np.testing.assert_allclose(ops.distill(z, ids, u, tail=True)[1], 0, atol=1e-15)
    np.testing.assert_allclose(ops.distill_gradient(z, ids, u, tail=True), 0, atol=1e-15)
    # by hand: p = (1/2, 1/2) against q = (1/2, 1/4): ln 2 / 2
    np.testing.assert_allclose(ops.distill(z[:1], ids[:1], np.zeros((1, 2)))[1], np.log(2) / 2)


def test_rows_that_leave_nothing():
    z = np.full((2, 4), -np.inf)
    z[1, 2] = 0.3
    assert ops.logprob(z, [1, 2]).tolist() == [-np.inf, 0.0]
    assert ops.entropy(z).tolist() == [0.0, 0.0]
    np.testing.assert_array_equal(ops.logprob_gradient(z, [1, 2], [1., 1.], [1., 1.]), 0)
    np.testing.assert_array_equal(
        ops.distill_gradient(z, [[1], [2]], [[-.1], [-.1]], tail=True, targets=[1, 2], ce=.5)[0], 0)


def test_top_order():
    z = np.array([[0.0, -0.0, 1.0, np.nan, 1.0, -np.inf]])
    assert ops.top(z, 6).tolist() == [[2, 4, 0, 1, 5, 3]]
