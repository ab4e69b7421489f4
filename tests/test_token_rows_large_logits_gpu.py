"""Token scoring and distillation on rows with finite masks and logits of any
size: masks from -1e9 to -1e30, rows whose every logit is one, ordinary logits
at very small temperatures.  Against the float64 oracle (oracle/token_ops.py).

Tolerances as in test_token_rows_gpu.py; where log q_r, the student's mass
outside the slots, is a large negative number, its term of the divergence is
off by 8 u of its size (three roundings of (z - m) / temperature, one of the
product, one of the sum, rounded up)."""
import numpy as np
import pytest

from oracle import token_ops as ops
from tests.helpers import Dev
from tests.test_token_rows_gpu import (NO, ROUND, U, Rows, check_score, check_score_gradient, distill, err_sum, logits,
                                       near, score, score_gradient)

pytestmark = pytest.mark.gpu

# a cluster, a CTA (several batches of a thread, and one) and a warp per row
SHAPES = [(6, 20001), (78, 9001), (6, 3001), (450, 600)]
MASKS = [-1e9, -1e10, -1e18, -1e20, -1e30]
TOP = 24


@pytest.fixture(scope="module")
def dev():
    return Dev()


def masked_rows(rng, rows, vocab, mask):
    """Six kinds of row: the first half masked, 99 % of it, all of it, all but
    one token, all but TOP tokens, half of it beside tokens at -inf."""
    z = logits(rng, rows, vocab)
    ids = np.stack([rng.choice(vocab, TOP, replace=False) for _ in range(rows)])
    for i in range(rows):
        kind = i % 6
        if kind == 0:
            z[i, :vocab // 2] = mask
        elif kind == 1:
            z[i, rng.random(vocab) < 0.99] = mask
        elif kind == 2:
            z[i] = mask
        elif kind == 3:
            z[i, np.arange(vocab) != vocab // 2] = mask
        elif kind == 4:
            z[i, np.setdiff1d(np.arange(vocab), ids[i])] = mask
        else:
            z[i, vocab // 2:] = mask
            z[i, ::3] = -np.inf
    return z, ids.astype(np.uint32)


def check_losses(z, got, ids, teacher, tau, tail, targets, kd, ce, scale):
    """check_distill of test_token_rows_gpu.py with the mass outside the slots
    by logarithms, so that it may be as small as e^(-1e30)."""
    args = dict(temperature=tau, tail=tail, targets=targets, kd=kd, ce=ce)
    p, inside, rest, _ = ops._slots(ids, teacher, z.shape[1], 1.0, tail)
    lq = ops.log_softmax(z.host, tau)
    q, size = np.exp(lq), np.where(np.isfinite(lq), np.abs(lq), 0.0)
    es = err_sum(z.shape[1])
    lp = np.where(p > 0, np.abs(np.log(np.where(p > 0, p, 1))), 0)
    e_p = 8 * U * (1 + np.abs(teacher).max(-1, keepdims=True))
    e_rest = (e_p[:, 0] + 140 * U) * (p.sum(-1) + rest) if tail else np.zeros(len(p))
    out = np.where(inside, -np.inf, lq)
    m = out.max(-1)
    share = np.where(np.isfinite(m)[:, None], np.exp(out - np.where(np.isfinite(m), m, 0)[:, None]), 0.0)
    sum_out = share.sum(-1)
    lq_r = np.where(np.isfinite(m), np.abs(np.where(np.isfinite(m), m, 0) + np.log(np.maximum(sum_out, 1))), 0)
    share = share / np.maximum(sum_out, 1)[:, None]
    log_rest = np.abs(np.log(np.maximum(np.maximum(rest, e_rest), 1e-30)))
    want_loss, want_kl = ops.distill(z.host, ids, teacher, **args)
    tol = (p * (2 * es + (e_p + 8 * U) * (1 + lp + size))).sum(-1) + e_rest * (2 + log_rest + lq_r) \
        + rest * (2 * es + 8 * U * (lq_r + log_rest)) + 16 * U
    if "kl" in got:
        near(got["kl"], want_kl, tol)
        l1 = ops.log_softmax(z.host)
        t1 = np.zeros(len(p))
        if targets is not None:
            t, ok = ops._given(targets, z.shape[1])
            t1 = np.where(ok, np.abs(l1[np.arange(len(t)), np.where(ok, t, 0)]), 0)
            t1 = np.where(np.isfinite(t1), t1, 0)
        near(got["loss"], want_loss, abs(kd) * tol + abs(ce) * (es + 8 * U * (t1 + 16))
             + 4 * U * np.where(np.isfinite(want_loss), np.abs(want_loss), 0))
    if "grad" in got:
        want = ops.distill_gradient(z.host, ids, teacher, row_scale=scale, **args)
        tol = abs(kd) / tau * (q * (2 * es + 8 * U * (np.minimum(size, 200) + 16)) + p * (e_p + 4 * U)
                               + share * (e_rest + rest * (2 * es + 8 * U * (16 + 200)))[:, None])
        if targets is not None and ce:
            l1 = ops.log_softmax(z.host)
            s1 = np.where(np.isfinite(l1), np.minimum(np.abs(l1), 200), 0)
            tol += abs(ce) * (np.exp(l1) * (2 * es + 8 * U * (s1 + 16)) + 4 * U * (want != 0))
        tol *= np.abs(scale)[:, None]
        near(got["grad"], want, tol + 2 * ROUND[z.type] * np.abs(want)
             + (2.0 ** -25 if z.type == "f16" else 2.0 ** -126))


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("rows,vocab", SHAPES)
@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("tau", [0.7, 1.0, 2.0, 4.0])
def test_scoring_finite_masks(dev, type, rows, vocab, mask, tau):
    rng = np.random.default_rng(31)
    tau = float(np.float32(tau))
    zh, _ = masked_rows(rng, rows, vocab, mask)
    z = Rows(dev, zh, type)
    targets = np.argmax(z.host, 1)
    got = score(dev, z, targets, 40, tau)
    check_score(z, got, targets, 40, tau)
    gl, ge = rng.standard_normal(rows).astype(np.float32), rng.standard_normal(rows).astype(np.float32)
    check_score_gradient(z, score_gradient(dev, z, targets, gl, ge, tau), targets, gl, ge, tau)


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("rows,vocab", SHAPES)
@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("tau", [0.7, 1.0, 2.0])
def test_distillation_finite_masks(dev, type, tail, rows, vocab, mask, tau):
    rng = np.random.default_rng(32)
    tau = float(np.float32(tau))
    zh, ids = masked_rows(rng, rows, vocab, mask)
    z = Rows(dev, zh, type)
    teacher = np.log(rng.dirichlet(np.ones(TOP), rows) * 0.95).astype(np.float32)
    targets = np.argmax(z.host, 1).astype(np.uint32)
    targets[::7] = NO
    scale = rng.uniform(0.2, 2, rows).astype(np.float32)
    args = dict(tau=tau, tail=tail, targets=targets, kd=0.8, ce=0.3)
    one = distill(dev, z, ids, teacher, **args)
    two = distill(dev, z, ids, teacher, "tl_distill_backward_rows", scale=scale, out=z.like(), stats=one["stats"], **args)
    both = distill(dev, z, ids, teacher, "tl_distill_train_rows", scale=scale, out=z.like(), **args)
    for got in (one, two, both):
        check_losses(z, got, ids, teacher, scale=scale, **args)


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab", SHAPES)
@pytest.mark.parametrize("tau", [1e-5, 1e-6, 1e-7, 1e-9, 1e-20, 1e-38])
def test_very_small_temperatures(dev, type, rows, vocab, tau):
    """Log probabilities of 1e6 to beyond fp32 (there -inf), entropies and
    gradients of rows that are all but one-hot."""
    rng = np.random.default_rng(33)
    z = Rows(dev, logits(rng, rows, vocab), type)
    # two tokens alike at the top of every other row
    z.view[::2, 5] = z.view[::2].amax(1)
    z.host = z.view.double().cpu().numpy()
    tau = float(np.float32(tau))
    targets = np.argmax(z.host, 1)
    got = score(dev, z, targets, 3, tau)
    lq = ops.log_softmax(z.host, tau)
    es = err_sum(vocab)
    near(got["logprob"], ops.logprob(z.host, targets, tau), es + 4 * U * 16)
    near(got["entropy"], ops.entropy(z.host, tau), 4 * es + 4 * U * 16)
    ids = ops.top(z.host, 3)
    np.testing.assert_array_equal(got["top_ids"], ids)
    with np.errstate(over="ignore"):
        want = np.take_along_axis(lq, ids, 1).astype(np.float32).astype(np.float64)
    near(got["top_logprob"], want, es + 4 * U * (np.where(np.isfinite(want), np.abs(want), 0) + 16))
    if tau >= 1e-20:  # 1 / tau times a gradient stays in fp32
        gl = np.full(rows, tau, np.float32)
        zero = np.zeros(rows, np.float32)
        check_score_gradient(z, score_gradient(dev, z, targets, gl, zero, tau), targets, gl, zero, tau)


@pytest.mark.parametrize("rows,vocab", SHAPES)
@pytest.mark.parametrize("base,tau", [(3e7, 2.0), (9e7, 8.0), (3e8, 32.0), (-3e8, 32.0), (1.5e8, 1.0), (-1.5e8, 1.0),
                                      (5e9, 512.0), (-5e9, 256.0), (1e20, 1e13), (1e30, 1e23), (-1e30, 1e23)])
def test_large_logits_that_differ(dev, rows, vocab, base, tau):
    """Logits next to one another far from 0: (z - m) / temperature of order 1
    where z / temperature is up to 2^24."""
    rng = np.random.default_rng(34)
    base, tau = float(np.float32(base)), float(np.float32(tau))
    unit = np.spacing(np.float32(abs(base)))
    zh = base + rng.integers(-6, 7, (rows, vocab)) * np.float64(unit)
    z = Rows(dev, zh)
    np.testing.assert_array_equal(z.host, zh)
    targets = rng.integers(0, vocab, rows)
    check_score(z, score(dev, z, targets, 20, tau), targets, 20, tau)
    one = np.ones(rows, np.float32)
    check_score_gradient(z, score_gradient(dev, z, targets, one, one, tau), targets, one, one, tau)
    ids = np.stack([rng.choice(vocab, TOP, replace=False) for _ in range(rows)]).astype(np.uint32)
    teacher = np.log(rng.dirichlet(np.ones(TOP), rows) * 0.9).astype(np.float32)
    for tail in (False, True):
        args = dict(tau=tau, tail=tail, targets=None, kd=tau, ce=0.0)
        got = distill(dev, z, ids, teacher, "tl_distill_train_rows", scale=one, out=z.like(), **args)
        check_losses(z, got, ids, teacher, scale=one, **args)
