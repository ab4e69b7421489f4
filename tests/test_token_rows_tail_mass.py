"""Distillation with the teacher's tail where the masses that the loss counts
do not add up to 1: slots of more than 1 together (no rest), and rows where
the student has no token outside the slots (the rest is dropped).  The
gradient is the derivative of the loss there too.  The oracle on the CPU
against central differences, the kernels against the oracle and against
differences of their own loss."""
import numpy as np
import pytest

from oracle import token_ops as ops
from tests.helpers import Dev
from tests.test_token_rows_gpu import ROUND, U, Rows, check_distill, distill, err_sum, near
from tests.test_token_rows_oracle import differences


@pytest.fixture(scope="module")
def dev():
    return Dev()


def rows_of(rng, rows, vocab, top):
    """Kinds of row, by 5: a teacher of ordinary mass; slots of more than 1;
    nothing outside the slots; both; no slots."""
    z = rng.standard_normal((rows, vocab)) * 2
    ids = np.stack([rng.choice(vocab, top, replace=False) for _ in range(rows)]).astype(np.uint32)
    teacher = np.log(rng.dirichlet(np.ones(top), rows) * 0.9)
    for i in range(rows):
        kind = i % 5
        if kind in (1, 3):
            teacher[i] = teacher[i] / 2
        if kind in (2, 3):
            z[i, np.setdiff1d(np.arange(vocab), ids[i])] = -np.inf
        if kind == 4:
            ids[i] = ops.NO_TOKEN
    return z, ids, teacher.astype(np.float32)


@pytest.mark.parametrize("temperature,teacher_temperature,ce", [(1.0, 1.0, 0.0), (2.0, 1.0, 0.3), (1.0, 2.0, 0.3)])
def test_oracle_gradient_against_differences(temperature, teacher_temperature, ce):
    """Step and tolerance as in test_token_rows_oracle.py."""
    rng = np.random.default_rng(41)
    z, ids, teacher = rows_of(rng, 5, 11, 3)
    # a row as an example: p = .5, .3, .15 at a teacher temperature of 2
    teacher[0] = np.log([.5, .3, .15])
    args = dict(temperature=temperature, teacher_temperature=teacher_temperature, tail=True,
                targets=ids[:, 0] % 11, kd=0.7, ce=ce)
    want = differences(lambda x: ops.distill(x, ids, teacher, **args)[0], z)
    np.testing.assert_allclose(ops.distill_gradient(z, ids, teacher, **args), want, atol=2e-9)


def check_gradient(z, got, ids, teacher, tau, teacher_tau, targets, kd, ce, scale):
    """The gradient's bounds in test_token_rows_gpu.py with the student's part
    P q in place of q, P the masses counted together: P times q's error, and q
    times P's, which is that of the rest (a float64 sum of the p's with e_p
    each, rounded once or twice)."""
    p, inside, rest, _ = ops._slots(ids, teacher, z.shape[1], teacher_tau, True)
    lq = ops.log_softmax(z.host, tau)
    q, size = np.exp(lq), np.where(np.isfinite(lq), np.abs(lq), 0.0)
    es = err_sum(z.shape[1])
    e_p = 8 * U * (1 + np.abs(teacher / teacher_tau).max(-1, keepdims=True))
    total = p.sum(-1, keepdims=True) + rest[:, None]
    e_rest = (e_p + 140 * U) * total
    out = np.where(inside, 0, q)
    q_r = out.sum(-1, keepdims=True)
    share = out / np.where(q_r > 0, q_r, 1)
    lq_r = np.where(q_r > 0, np.abs(np.log(np.where(q_r > 0, q_r, 1))), 0.0)
    want = ops.distill_gradient(z.host, ids, teacher, temperature=tau, teacher_temperature=teacher_tau, tail=True,
                                targets=targets, kd=kd, ce=ce, row_scale=scale)
    tol = kd / tau * (q * (total * (2 * es + 8 * U * (size + 16)) + e_rest) + p * (e_p + 4 * U)
                      + share * (e_rest + rest[:, None] * (2 * es + 8 * U * (16 + lq_r))))
    if ce:
        l1 = ops.log_softmax(z.host)
        s1 = np.where(np.isfinite(l1), np.abs(l1), 0)
        tol += ce * (np.exp(l1) * (2 * es + 8 * U * (s1 + 16)) + 4 * U * (want != 0))
    near(got, want, tol * scale[:, None] + 2 * ROUND[z.type] * np.abs(want)
         + (2.0 ** -25 if z.type == "f16" else 2.0 ** -126))


# a cluster, a CTA and a warp per row
SHAPES = [(5, 20001), (5, 3001), (450, 600)]


@pytest.mark.gpu
@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab", SHAPES)
@pytest.mark.parametrize("tau,teacher_tau,ce", [(1.0, 1.0, 0.0), (1.0, 2.0, 0.3), (2.0, 1.0, 0.3), (0.5, 4.0, 0.0)])
def test_kernels_against_the_oracle(dev, type, rows, vocab, tau, teacher_tau, ce):
    rng = np.random.default_rng(42)
    z, ids, teacher = rows_of(rng, rows, vocab, 24)
    z = Rows(dev, z, type)
    targets = ids[:, 1] % vocab if ce else None
    scale = rng.uniform(0.5, 1.5, rows).astype(np.float32)
    args = dict(tau=tau, teacher_tau=teacher_tau, targets=targets, kd=0.8, ce=ce)
    one = distill(dev, z, ids, teacher, tail=True, **args)
    check_distill(z, one, ids, teacher, tail=True, **args)
    two = distill(dev, z, ids, teacher, "tl_distill_backward_rows", tail=True, scale=scale, out=z.like(),
                  stats=one["stats"], **args)
    both = distill(dev, z, ids, teacher, "tl_distill_train_rows", tail=True, scale=scale, out=z.like(), **args)
    for k in ("loss", "kl"):
        np.testing.assert_array_equal(both[k], one[k])
    for got in (two, both):
        check_gradient(z, got["grad"], ids, teacher, scale=scale, **args)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab", SHAPES)
def test_kernels_against_differences(dev, rows, vocab):
    """As test_gradients_against_differences in test_token_rows_gpu.py.  The
    loss is at most 10 times as large here (P <= 10) and so are its third
    derivative and its rounding: 5e-3."""
    rng = np.random.default_rng(43)
    zh, ids, teacher = rows_of(rng, rows, vocab, 24)
    zh = zh.astype(np.float32)
    h, way = 1e-2, rng.standard_normal(zh.shape).astype(np.float32)
    args = dict(tail=True, targets=ids[:, 1] % vocab, ce=0.4, kd=0.9, tau=1.5, teacher_tau=1.5)
    grad = distill(dev, Rows(dev, zh), ids, teacher, "tl_distill_train_rows", out=Rows(dev, zh).like(), **args)["grad"]
    ends = [distill(dev, Rows(dev, zh + s * h * way), ids, teacher, **args)["loss"].astype(np.float64)
            for s in (1, -1)]
    np.testing.assert_allclose((grad * way).sum(-1), (ends[0] - ends[1]) / (2 * h), atol=5e-3)


@pytest.mark.gpu
def test_ordinary_rows_keep_their_statistics(dev):
    """Where the masses add up to 1 the statistics' last place is 0."""
    rng = np.random.default_rng(44)
    for rows, vocab in SHAPES:
        z, ids, teacher = rows_of(rng, rows, vocab, 24)
        z = Rows(dev, z)
        for tail in (False, True):
            st = dev.host(distill(dev, z, ids, teacher, tail=tail)["stats"])
            assert not st[0::5, 7].any() and not st[4::5, 7].any()
            if not tail:
                assert not st[:, 7].any()
