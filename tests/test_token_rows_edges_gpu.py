"""Token scoring and distillation at single edges of what the entry points
accept, against the float64 oracle (oracle/token_ops.py)."""
import ctypes
import threading

import numpy as np
import pytest

from oracle import token_ops as ops
from templit_b200 import capi
from tests.helpers import Dev
from tests.test_token_rows_gpu import (U, Rows, all_three, base_desc, distill, f32, ids_of,
                                       near, score, teacher_of, u32)

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


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("rows,vocab", SHAPES)
@pytest.mark.parametrize("tau", [0.25, 0.5, 0.7, 1.0, 2.0])
@pytest.mark.parametrize("tail", [False, True])
def test_losses_of_masks_at_the_lowest_value(dev, type, rows, vocab, tau, tail):
    """A slot of probability p at the type's lowest value L: p (-L) / tau is
    the divergence to a part in 10^37, beyond fp32 (+inf) or not; so is the
    rest's where every token outside the slots is at L.  A term's error is
    that of p, 8 u (1 + |log p|), and 8 u more."""
    rng = np.random.default_rng(52)
    low = {"f32": -3.4028234663852886e38, "bf16": -3.3895313892515355e38}[type]
    tau = float(np.float32(tau))
    ids = np.stack([rng.choice(vocab, 9, replace=False) for _ in range(rows)]).astype(np.uint32)
    teacher = np.log(np.tile([.3, .2, .1, .1, .05, .05, .02, .01, 1e-35], (rows, 1))).astype(np.float32)
    z = rng.standard_normal((rows, vocab))
    for i in range(rows):
        if i % 4 == 0:
            z[i, ids[i, 8]] = low      # p = 1e-35: a divergence of some 1000
        elif i % 4 == 1:
            z[i, ids[i, 0]] = low      # p = 0.3
        elif i % 4 == 2:
            z[i, np.setdiff1d(np.arange(vocab), ids[i])] = low
        else:
            z[i] = low
    z = Rows(dev, z, type)
    want_loss, want_kl = ops.distill(z.host, ids, teacher, temperature=tau, tail=tail, kd=0.5)
    with np.errstate(over="ignore"):
        want_loss, want_kl = (w.astype(np.float32).astype(np.float64) for w in (want_loss, want_kl))
    for name, out in (("tl_distill_rows", None), ("tl_distill_train_rows", z.like())):
        got = distill(dev, z, ids, teacher, name, tau=tau, tail=tail, kd=0.5, out=out)
        for k, want in (("kl", want_kl), ("loss", want_loss)):
            tol = 8 * U * (2 + 81) * (20 + np.where(np.isfinite(want), np.abs(want), 0))
            near(got[k], want, tol)


def test_vocabularies_on_two_host_threads(dev):
    """Calls of two vocabularies that need different amounts of shared memory,
    from two host threads on a stream each: none may fail or change another's
    result."""
    torch, rng = dev.torch, np.random.default_rng(53)
    plans = []
    for vocab in (1 << 20, 500000):
        z = Rows(dev, rng.standard_normal((1, vocab)))
        ids = rng.choice(vocab, 16, replace=False)[None].astype(np.uint32)
        teacher = np.log(np.full((1, 16), 0.05)).astype(np.float32)
        want = distill(dev, z, ids, teacher, tail=True)["loss"]
        held = [z, u32(dev, ids), f32(dev, teacher), dev.empty((1,)), torch.cuda.Stream()]
        d = base_desc(capi.TlDistillDesc, dev, z, 1.0)
        d.teacher_temperature, d.tail, d.top, d.kd_weight = 1.0, 1, 16, 1.0
        d.teacher_ids, d.teacher, d.loss = held[1].data_ptr(), held[2].data_ptr(), held[3].data_ptr()
        plans.append((d, held, want))
    torch.cuda.synchronize()
    failed = []

    def work(d, stream):
        ref, raw = ctypes.byref(d), ctypes.c_void_p(stream.cuda_stream)
        for _ in range(3000):
            if dev.lib.tl_distill_rows(ref, raw) != capi.TL_OK:
                failed.append(dev.lib.tl_last_error())
                return

    threads = [threading.Thread(target=work, args=(d, held[-1])) for d, held, _ in plans]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed, failed
    for d, held, want in plans:
        np.testing.assert_array_equal(dev.host(held[3]), want)


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab,offset", [(1 << 20, 0), ((1 << 20) - 3, 3)])
def test_the_longest_vocabularies_of_the_tail(dev, type, vocab, offset):
    """A bit per token up to TL_DISTILL_MAX_VOCAB, slots at both ends."""
    rng = np.random.default_rng(54)
    z = Rows(dev, rng.standard_normal((2, vocab)), type, offset=offset)
    ids = np.stack([np.concatenate([[0, 1, vocab - 1, vocab - 2], 2 + rng.choice(vocab - 4, 60, replace=False)])
                    for _ in range(2)]).astype(np.uint32)
    teacher = np.log(rng.dirichlet(np.ones(64), 2) * 0.9).astype(np.float32)
    all_three(dev, z, ids, teacher, np.array([1, 2], np.float32), tail=True, targets=np.array([vocab - 1, 77]), ce=0.5,
              tau=2.0)


def test_calls_on_two_streams_at_once(dev):
    """Long calls that overlap on two streams give what each gives alone."""
    torch, rng = dev.torch, np.random.default_rng(55)
    jobs = []
    for seed in range(2):
        zt, ids, teacher = teacher_of(rng, 300, 30000, 32)
        jobs.append((Rows(dev, zt + rng.standard_normal(zt.shape), "bf16"), ids, teacher, torch.cuda.Stream()))
    args = dict(tail=True, targets=None, tau=2.0)
    alone = [distill(dev, z, ids, teacher, "tl_distill_train_rows", out=z.like(), **args) for z, ids, teacher, _ in jobs]
    alone_score = [score(dev, z, None, 30) for z, *_ in jobs]
    descs = []
    for z, ids, teacher, stream in jobs:
        out, loss = z.like(), dev.empty((300,))
        tops = [dev.empty((300, 30)), dev.empty((300, 30), torch.int32)]
        held = [u32(dev, ids), f32(dev, teacher), out, loss, tops]
        d = base_desc(capi.TlDistillDesc, dev, z, 2.0)
        d.teacher_temperature, d.tail, d.top, d.kd_weight = 1.0, 1, 32, 1.0
        d.teacher_ids, d.teacher, d.loss = held[0].data_ptr(), held[1].data_ptr(), loss.data_ptr()
        d.dlogits, d.d_row_stride = out.ptr(), out.stride
        s = base_desc(capi.TlTokenLogprobDesc, dev, z, 1.0)
        s.top, s.top_logprob, s.top_ids = 30, tops[0].data_ptr(), tops[1].data_ptr()
        descs.append((d, s, held, ctypes.c_void_p(stream.cuda_stream)))
    torch.cuda.synchronize()
    for _ in range(20):
        for d, s, _, raw in descs:
            capi.check(dev.lib.tl_distill_train_rows(ctypes.byref(d), raw), dev.lib, "tl_distill_train_rows")
            capi.check(dev.lib.tl_token_logprob_rows(ctypes.byref(s), raw), dev.lib, "tl_token_logprob_rows")
    torch.cuda.synchronize()
    for (_, _, held, _), one, tops in zip(descs, alone, alone_score):
        np.testing.assert_array_equal(held[2].get(), one["grad"])
        np.testing.assert_array_equal(dev.host(held[3]), one["loss"])
        np.testing.assert_array_equal(dev.host(held[4][0]), tops["top_logprob"])
        np.testing.assert_array_equal(ids_of(dev, held[4][1]), tops["top_ids"])
