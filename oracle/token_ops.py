"""Token scoring and distillation in float64 numpy, from their formulas:
the oracle of tl_token_logprob_rows, tl_distill_rows and their gradients
(include/templit_cuda.h).  Rows of logits are [rows, vocab]; -inf is a token
that cannot occur.  No counterpart in the reference, whose cross entropy
(src/my_metal/runtime.cpp:768-841) is its only operator on logits."""
from __future__ import annotations

import numpy as np

NO_TOKEN = 0xFFFFFFFF


def log_softmax(z, temperature=1.0):
    """Row log softmax of z / temperature; a row of -inf stays -inf."""
    x = np.asarray(z, np.float64) / temperature
    m = x.max(-1, keepdims=True)
    with np.errstate(divide="ignore", invalid="ignore"):
        d = np.where(np.isneginf(m), -np.inf, x - m)
        return np.where(np.isneginf(m), -np.inf, d - np.log(np.exp(d).sum(-1, keepdims=True)))


def _q_log_q(lq):
    return np.where(np.isneginf(lq), 0.0, np.exp(lq) * np.where(np.isneginf(lq), 0.0, lq))


def _given(targets, vocab):
    t = np.asarray(targets, np.uint32).astype(np.int64)
    return t, t < vocab


def logprob(z, targets, temperature=1.0):
    t, ok = _given(targets, z.shape[1])
    lq = log_softmax(z, temperature)
    return np.where(ok, lq[np.arange(len(t)), np.where(ok, t, 0)], 0.0)


def entropy(z, temperature=1.0):
    return -_q_log_q(log_softmax(z, temperature)).sum(-1)


def stats(z, temperature=1.0):
    z = np.asarray(z, np.float64)
    m = z.max(-1)
    with np.errstate(invalid="ignore"):
        d = np.where(np.isneginf(m)[:, None], -np.inf, (z - m[:, None]) / temperature)
    return np.stack([m, np.exp(d).sum(-1)], -1)


def top(z, k):
    """Ids of the k largest logits of each row, the lower id first among
    equals (0 and -0 alike), NaN last."""
    z = np.asarray(z, np.float64)
    nan = np.isnan(z)
    # numpy sorts by the last key first: not-NaN, value, index
    ids = np.broadcast_to(np.arange(z.shape[1]), z.shape)
    order = np.lexsort((ids, -np.where(nan, 0.0, z), nan), axis=-1)
    return order[:, :k]


def logprob_gradient(z, targets, d_logprob, d_entropy, temperature=1.0):
    """d (sum d_logprob * logprob + d_entropy * entropy) / dz."""
    lq = log_softmax(z, temperature)
    q = np.exp(lq)
    g = np.zeros_like(q)
    empty = np.isneginf(lq).all(-1)
    if d_logprob is not None:
        t, ok = _given(targets, z.shape[1])
        w = np.where(ok & ~empty, np.asarray(d_logprob, np.float64), 0.0)
        g -= w[:, None] * q
        g[np.arange(len(t)), np.where(ok, t, 0)] += w
    if d_entropy is not None:
        h = -_q_log_q(lq).sum(-1, keepdims=True)
        g -= np.asarray(d_entropy, np.float64)[:, None] * (_q_log_q(lq) + q * h)
    return g / temperature


def _slots(ids, teacher, vocab, teacher_temperature, tail):
    """[rows, vocab] p, [rows, vocab] membership and the rest of the mass."""
    ids = np.asarray(ids, np.uint32).astype(np.int64)
    u = np.asarray(teacher, np.float64) / teacher_temperature
    ok = (ids < vocab) & ~np.isneginf(u)
    rows = np.arange(len(ids))
    p = np.zeros((len(ids), vocab))
    inside = np.zeros((len(ids), vocab), bool)
    u = np.where(ok, u, -np.inf)
    some = ok.any(-1)
    if tail:
        w = np.exp(u)
        rest = np.where(some, np.maximum(0.0, 1.0 - w.sum(-1)), 0.0)
    else:
        m = np.where(some, u.max(-1), 0.0)
        w = np.exp(u - m[:, None])
        w = w / np.where(some, w.sum(-1), 1.0)[:, None]
        rest = np.zeros(len(ids))
    for k in range(ids.shape[1]):
        sel = ok[:, k]
        p[rows[sel], ids[sel, k]] = w[sel, k]
        inside[rows[sel], ids[sel, k]] = True
    return p, inside, rest, some


def distill(z, ids, teacher, temperature=1.0, teacher_temperature=1.0, tail=False, targets=None,
            kd=1.0, ce=0.0):
    """(loss, kl) per row."""
    p, inside, rest, _ = _slots(ids, teacher, z.shape[1], teacher_temperature, tail)
    lq = log_softmax(z, temperature)
    with np.errstate(divide="ignore", invalid="ignore"):
        kl = np.where(p > 0, p * (np.log(np.where(p > 0, p, 1.0)) - lq), 0.0).sum(-1)
        if tail:
            # q_r by logarithms, so that a small share outside the slots stays
            out = np.where(inside, -np.inf, lq)
            m = out.max(-1)
            has = ~np.isneginf(m)
            m0 = np.where(has, m, 0.0)
            lq_r = m0 + np.log(np.where(has, np.exp(out - m0[:, None]).sum(-1), 1.0))
            kl += np.where(has & (rest > 0), rest * (np.log(np.where(rest > 0, rest, 1.0)) - lq_r), 0.0)
    loss = kd * kl if kd else np.zeros_like(kl)
    if targets is not None and ce:
        t, ok = _given(targets, z.shape[1])
        nll = -log_softmax(z)[np.arange(len(t)), np.where(ok, t, 0)]
        loss = loss + np.where(ok, ce * np.where(ok, nll, 0.0), 0.0)
    return loss, kl


def distill_gradient(z, ids, teacher, temperature=1.0, teacher_temperature=1.0, tail=False,
                     targets=None, kd=1.0, ce=0.0, row_scale=None):
    """row_scale * d loss / dz."""
    p, inside, rest, some = _slots(ids, teacher, z.shape[1], teacher_temperature, tail)
    lq = log_softmax(z, temperature)
    empty = np.isneginf(lq).all(-1)
    q = np.exp(lq)
    total = p.sum(-1, keepdims=True)  # the masses that the loss counts: 1, or what a row has
    if tail:
        out = np.where(inside, -np.inf, lq)
        m = out.max(-1, keepdims=True)
        has = ~np.isneginf(m)
        total = total + np.where(has, rest[:, None], 0.0)
    g = np.where(some[:, None], total * q - p, 0.0)
    if tail:
        e = np.exp(np.where(has, out - np.where(has, m, 0.0), -np.inf))
        share = e / np.where(has, e.sum(-1, keepdims=True), 1.0)  # q_j / q_r
        g -= rest[:, None] * share
    g *= kd / temperature
    if targets is not None and ce:
        t, ok = _given(targets, z.shape[1])
        h = np.exp(log_softmax(z))
        h[np.arange(len(t)), np.where(ok, t, 0)] -= 1.0
        g += ce * np.where(ok[:, None], h, 0.0)
    g[empty] = 0.0
    return g if row_scale is None else g * np.asarray(row_scale, np.float64)[:, None]
