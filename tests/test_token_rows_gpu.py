"""Token scoring and distillation kernels (tl_token_logprob_rows,
tl_distill_rows and their gradients) against the float64 oracle
(oracle/token_ops.py) on the inputs as the kernels hold them.

Tolerances, from the arithmetic (u = 2^-24, fp32's rounding):
  a term e^x of a sum has the error of the exponential, 2^-22, and of its
  argument, 4 u |x|, where |x| e^x < 1: below 2^-20 together; a sum of V
  terms over at least 32 accumulators adds (V / 32 + 16) u.  SUM(V) is both.
  log q: SUM(V) + 4 u (|x| + 16).  H and KL: the sum's error on each term,
  and 4 u of the sum of the terms' sizes.  A gradient element: the error of
  q in each term it consists of, and half a unit of the logits' type (2^-11
  for fp16, with 2^-25 below its normal range; 2^-8 for bf16).
Ids are exact."""
import ctypes

import numpy as np
import pytest

from oracle import token_ops as ops
from templit_b200 import capi
from tests.helpers import Dev

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"f32": capi.TL_FLOAT32, "f16": capi.TL_FLOAT16, "bf16": capi.TL_BFLOAT16}
ROUND = {"f32": U, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
NO = ops.NO_TOKEN
GUARD = 7.0  # what the gaps between padded rows hold


def err_sum(vocab):
    return 2.0 ** -20 + (vocab / 32 + 16) * U


@pytest.fixture(scope="module")
def dev():
    return Dev()


def torch_type(dev, type):
    return {"f32": dev.torch.float32, "f16": dev.torch.float16, "bf16": dev.torch.bfloat16}[type]


class Rows:
    """Logits on the device, rows `stride` apart and `offset` elements into
    their buffer, and the same numbers in float64."""

    def __init__(self, dev, z, type="f32", pad=0, offset=0):
        rows, vocab = z.shape
        self.dev, self.type, self.stride, self.shape, self.offset = dev, type, vocab + pad, z.shape, offset
        dt = torch_type(dev, type)
        self.buf = dev.torch.full((offset + rows * self.stride + 8,), GUARD, dtype=dt, device=dev.dev)
        self.view = self.buf[offset:offset + rows * self.stride].view(rows, self.stride)[:, :vocab]
        self.view.copy_(dev.torch.from_numpy(z))
        self.host = self.view.double().cpu().numpy()

    def like(self, pad=None, offset=None):
        out = Rows.__new__(Rows)
        rows, vocab = self.shape
        out.dev, out.type, out.shape = self.dev, self.type, self.shape
        out.offset = self.offset if offset is None else offset
        out.stride = self.stride if pad is None else vocab + pad
        out.buf = self.dev.torch.full((out.offset + rows * out.stride + 8,), GUARD, dtype=self.buf.dtype,
                                      device=self.dev.dev)
        out.view = out.buf[out.offset:out.offset + rows * out.stride].view(rows, out.stride)[:, :vocab]
        return out

    def ptr(self):
        return self.buf.data_ptr() + self.offset * self.buf.element_size()

    def get(self):
        self.dev.torch.cuda.synchronize()
        return self.view.double().cpu().numpy()

    def untouched(self):
        """Whether everything outside the rows still holds GUARD."""
        keep = self.buf.clone()
        rows, vocab = self.shape
        keep[self.offset:self.offset + rows * self.stride].view(rows, self.stride)[:, :vocab] = GUARD
        return bool((keep == GUARD).all())


def u32(dev, a):
    return dev.torch.from_numpy(np.ascontiguousarray(np.asarray(a, np.uint32)).view(np.int32)).to(dev.dev)


def f32(dev, a):
    return dev.torch.from_numpy(np.ascontiguousarray(a, np.float32)).to(dev.dev)


def ids_of(dev, t):
    return dev.host(t).view(np.uint32).astype(np.int64)


def call(dev, name, desc):
    dev.call(name, ctypes.byref(desc), dev.stream)


def base_desc(cls, dev, z, tau):
    d = cls()
    d.logits, d.row_stride, d.type = z.ptr(), z.stride, TYPES[z.type]
    d.rows, d.vocab, d.temperature = z.shape[0], z.shape[1], tau
    return d


def score(dev, z, targets=None, top=0, tau=1.0):
    rows = z.shape[0]
    d = base_desc(capi.TlTokenLogprobDesc, dev, z, tau)
    d.top = top
    out = {"entropy": dev.empty((rows,)), "stats": dev.empty((rows, 2))}
    if targets is not None:
        t = u32(dev, targets)
        out["logprob"] = dev.empty((rows,))
        d.targets, d.logprob = t.data_ptr(), out["logprob"].data_ptr()
    if top:
        out["top_logprob"] = dev.empty((rows, top))
        out["top_ids"] = dev.empty((rows, top), dev.torch.int32)
        d.top_logprob, d.top_ids = out["top_logprob"].data_ptr(), out["top_ids"].data_ptr()
    d.entropy, d.stats = out["entropy"].data_ptr(), out["stats"].data_ptr()
    call(dev, "tl_token_logprob_rows", d)
    return {k: ids_of(dev, v) if k == "top_ids" else dev.host(v) for k, v in out.items()}


def near(got, want, tol):
    """|got - want| <= tol where want is finite, equal where not."""
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    fin = np.isfinite(want)
    np.testing.assert_array_equal(got[~fin], want[~fin])
    assert np.isfinite(got[fin]).all()
    over = np.abs(got - want)[fin] - np.broadcast_to(tol, want.shape)[fin]
    assert over.size == 0 or over.max() <= 0, (over.max(), np.abs(got - want)[fin].max())


def check_score(z, got, targets, top, tau):
    vocab = z.shape[1]
    es = err_sum(vocab)
    lq = ops.log_softmax(z.host, tau)
    size = np.where(np.isfinite(lq), np.abs(lq), 0.0)
    if targets is not None:
        want = ops.logprob(z.host, targets, tau)
        near(got["logprob"], want, es + 4 * U * (np.where(np.isfinite(want), np.abs(want), 0) + 16))
    want = ops.entropy(z.host, tau)
    near(got["entropy"], want, 2 * es * (1 + (np.exp(lq) * size).sum(-1)) + 4 * U * 16)
    st = ops.stats(z.host, tau)
    np.testing.assert_array_equal(got["stats"][:, 0], st[:, 0])
    near(got["stats"][:, 1], st[:, 1], es * st[:, 1])
    if top:
        ids = ops.top(z.host, top)
        np.testing.assert_array_equal(got["top_ids"], ids)
        want = np.take_along_axis(lq, ids, 1)
        near(got["top_logprob"], want, es + 4 * U * (np.where(np.isfinite(want), np.abs(want), 0) + 16))


def logits(rng, rows, vocab, sharp=3.0):
    return rng.standard_normal((rows, vocab)) * rng.uniform(0.3, sharp, (rows, 1)) + rng.uniform(-5, 5, (rows, 1))


SIZES = [(1, 1), (3, 2), (2, 7), (5, 31), (4, 33), (3, 200), (7, 511), (5, 1023), (6, 2047), (300, 2048), (5, 2049),
         (3, 4096), (4, 4100), (3, 6001), (3, 8192), (4, 8193), (2, 16411), (3, 32768), (3, 50001), (2, 65536),
         (2, 131072), (1, 200003), (1, 2048), (160, 40000)]
# many rows, some of them short enough for a warp each
SIZES += [(900, 2500), (900, 4093), (900, 8000)]
SIZES += [(700, v) for v in (1, 6, 30, 129, 511, 512, 1000, 1026, 2047, 2048, 2050, 4095, 4096, 4099)]


def repeat(many, *arrays):
    """The rows many times over: enough of them to take a warp each."""
    out = [a if a is None or not many else np.concatenate([a] * (-(-900 // len(a)))) for a in arrays]
    return out if len(out) > 1 else out[0]


@pytest.mark.parametrize("type", list(TYPES))
@pytest.mark.parametrize("rows,vocab", SIZES)
def test_scoring_sizes(dev, type, rows, vocab):
    rng = np.random.default_rng(rows * 1000003 + vocab)
    z = Rows(dev, logits(rng, rows, vocab), type)
    top = min(vocab, int(rng.integers(1, 129)))
    targets = rng.integers(0, vocab, rows)
    check_score(z, score(dev, z, targets, top), targets, top, 1.0)


@pytest.mark.parametrize("type", list(TYPES))
@pytest.mark.parametrize("rows", [9, 700])
@pytest.mark.parametrize("vocab,pad,offset", [(2048, 8, 0), (2048, 1, 3), (50001, 0, 1), (50001, 7, 5), (777, 3, 2),
                                              (9001, 0, 1), (40, 2, 1), (131075, 0, 3)])
def test_scoring_strides_and_alignment(dev, type, vocab, pad, offset, rows):
    rows = min(rows, 9 if vocab > 4200 else rows)
    rng = np.random.default_rng(vocab + pad)
    z = Rows(dev, logits(rng, rows, vocab), type, pad, offset)
    targets = rng.integers(0, vocab, rows)
    check_score(z, score(dev, z, targets, 20, 0.7), targets, 20, 0.7)
    assert z.untouched()


@pytest.mark.parametrize("top", [1, 2, 3, 5, 31, 32, 33, 64, 127, 128])
@pytest.mark.parametrize("vocab", [128, 2048, 3000, 50001])
def test_scoring_alternatives(dev, top, vocab):
    rng = np.random.default_rng(top)
    z = Rows(dev, logits(rng, 6, vocab), "bf16")
    check_score(z, score(dev, z, None, top, 2.5), None, top, 2.5)


@pytest.mark.parametrize("type", list(TYPES))
@pytest.mark.parametrize("vocab,many", [(130, False), (2048, False), (5000, False), (70001, False),
                                        (130, True), (512, True), (2047, True), (2048, True), (4001, True)])
def test_scoring_ties_and_order(dev, type, vocab, many):
    """Equal rows, two values, ascending, descending, all in one place, zeros
    of both signs: the lowest ids first among equals, and more candidates
    than any buffer of a fast path can expect."""
    rng = np.random.default_rng(5)
    z = np.zeros((9, vocab))
    z[0] = 1.5
    z[1] = rng.integers(0, 2, vocab)
    z[2] = np.arange(vocab) / vocab
    z[3] = -np.arange(vocab) / vocab
    z[4, :128] = np.arange(128) + 1
    z[5, -128:] = np.arange(128) + 1
    z[6] = np.where(rng.integers(0, 2, vocab), 0.0, -0.0)
    z[7, ::64] = 2.0
    z[8] = np.floor(rng.standard_normal(vocab) * 2)
    z = Rows(dev, repeat(many, z), type)
    targets = np.full(len(z.host), vocab - 1)
    for top in (128, 40):
        check_score(z, score(dev, z, targets, top), targets, top, 1.0)


@pytest.mark.parametrize("type", list(TYPES))
@pytest.mark.parametrize("vocab,many", [(129, False), (2048, False), (20001, False), (100000, False),
                                        (129, True), (1030, True), (2048, True), (4001, True)])
def test_scoring_masks(dev, type, vocab, many):
    """Masked tokens: -inf, the type's lowest value, rows with one token, and
    with none."""
    rng = np.random.default_rng(6)
    low = {"f32": -3.4028234663852886e38, "f16": -65504.0, "bf16": -3.3895313892515355e38}[type]
    z = logits(rng, 8, vocab)
    z[0, rng.random(vocab) < 0.5] = -np.inf
    z[1, rng.random(vocab) < 0.5] = low
    z[2] = -np.inf
    z[3] = low
    z[4] = -np.inf
    z[4, vocab // 2] = 3.0
    z[5, 1:] = low
    z[6, :-1] = -np.inf
    z[7, :vocab // 2] = -np.inf
    z, targets = repeat(many, z, np.array([0, 1, 2, 3, vocab // 2, 0, vocab - 1, 5]))
    z = Rows(dev, z, type)
    top = min(vocab, 64)
    got = score(dev, z, targets, top)
    check_score(z, got, targets, top, 1.0)
    assert got["entropy"][2] == 0 and got["logprob"][2] == -np.inf


@pytest.mark.parametrize("vocab,many", [(100, False), (2048, False), (30001, False), (100, True), (2048, True)])
def test_scoring_nan_and_infinity(dev, vocab, many):
    rng = np.random.default_rng(7)
    z = logits(rng, 4, vocab)
    z[0, 3] = np.nan
    z[1, 50] = np.inf
    z[2] = np.nan
    z, targets = repeat(many, z, np.array([0, 1, 2, 3]))
    zr = Rows(dev, z)
    got = score(dev, zr, targets, 100)
    assert np.isnan(got["logprob"][:3]).all() and np.isnan(got["entropy"][:3]).all()
    assert np.isnan(got["top_logprob"][:3]).all()
    np.testing.assert_array_equal(got["top_ids"], ops.top(zr.host, 100))
    assert np.isfinite(got["logprob"][3]) and np.isfinite(got["entropy"][3])


def test_scoring_given_tokens(dev):
    rng = np.random.default_rng(8)
    z = Rows(dev, logits(rng, 4, 300))
    targets = np.array([7, NO, 299, 300], np.uint32)
    assert dev.status() == 0
    got = score(dev, z, targets)
    near(got["logprob"], [ops.logprob(z.host, targets)[0], 0, ops.logprob(z.host, targets)[2], 0], 1e-5)
    assert dev.status() == capi.TL_FLAG_INDEX_RANGE
    score(dev, z, np.array([0, NO, NO, 299], np.uint32))
    assert dev.status() == 0


def test_scoring_single_outputs(dev):
    """Each output alone equals the one of a full call, bit for bit, and
    again on a second call."""
    rng = np.random.default_rng(9)
    for type, vocab, rows in (("f32", 2048, 40), ("bf16", 50001, 5), ("f16", 9000, 2), ("f32", 2048, 700)):
        z = Rows(dev, logits(rng, rows, vocab), type)
        targets = rng.integers(0, vocab, rows)
        full = score(dev, z, targets, 17, 1.3)
        again = score(dev, z, targets, 17, 1.3)
        for k in full:
            np.testing.assert_array_equal(full[k], again[k])
        t = u32(dev, targets)
        for name in ("entropy", "stats", "logprob", "top"):
            d = base_desc(capi.TlTokenLogprobDesc, dev, z, 1.3)
            o = dev.empty((rows, {"stats": 2, "top": 17}.get(name, 1)))
            i = dev.empty((rows, 17), dev.torch.int32)
            if name == "top":
                d.top, d.top_logprob, d.top_ids = 17, o.data_ptr(), i.data_ptr()
            else:
                setattr(d, name, o.data_ptr())
            if name == "logprob":
                d.targets = t.data_ptr()
            call(dev, "tl_token_logprob_rows", d)
            if name == "top":
                np.testing.assert_array_equal(ids_of(dev, i), full["top_ids"])
                np.testing.assert_array_equal(dev.host(o), full["top_logprob"])
            else:
                np.testing.assert_array_equal(dev.host(o).reshape(full[name].shape), full[name])


# ------------------------------------------------------- gradient of scoring

def score_gradient(dev, z, targets, gl, ge, tau=1.0, out=None):
    rows = z.shape[0]
    kept = {"e": dev.empty((rows,)), "s": dev.empty((rows, 2))}
    d = base_desc(capi.TlTokenLogprobDesc, dev, z, tau)
    d.entropy, d.stats = kept["e"].data_ptr(), kept["s"].data_ptr()
    call(dev, "tl_token_logprob_rows", d)
    t = u32(dev, targets)
    held = [t]
    d.targets = t.data_ptr()
    for name, g in (("d_logprob", gl), ("d_entropy", ge)):
        if g is not None:
            held.append(f32(dev, g))
            setattr(d, name, held[-1].data_ptr())
    out = out or z.like()
    d.dlogits, d.d_row_stride = out.ptr(), out.stride
    call(dev, "tl_token_logprob_backward_rows", d)
    return out.get()


def check_score_gradient(z, got, targets, gl, ge, tau):
    want = ops.logprob_gradient(z.host, targets, gl, ge, tau)
    lq = ops.log_softmax(z.host, tau)
    q, size = np.exp(lq), np.where(np.isfinite(lq), np.abs(lq), 0.0)
    eq = 2 * err_sum(z.shape[1]) + 4 * U * (size + 16)
    h = ops.entropy(z.host, tau)[:, None]
    scale = np.zeros((z.shape[0], 1))
    tol = np.zeros_like(q)
    if gl is not None:
        tol += np.abs(gl)[:, None] * q * eq + 4 * U * np.abs(gl)[:, None] * (want != 0)
        scale = scale + np.abs(gl)[:, None]
    if ge is not None:
        tol += np.abs(ge)[:, None] * q * (eq * (size + h + 2) + 8 * U * 16)
    tol = tol / tau + 2 * ROUND[z.type] * np.abs(want) + (2.0 ** -25 if z.type == "f16" else 2.0 ** -126)
    near(got, want, tol)


@pytest.mark.parametrize("type", list(TYPES))
@pytest.mark.parametrize("rows,vocab", SIZES)
def test_scoring_gradient_sizes(dev, type, rows, vocab):
    rng = np.random.default_rng(rows * 7 + vocab)
    z = Rows(dev, logits(rng, rows, vocab), type)
    targets = rng.integers(0, vocab, rows)
    gl, ge = rng.standard_normal(rows).astype(np.float32), rng.standard_normal(rows).astype(np.float32)
    check_score_gradient(z, score_gradient(dev, z, targets, gl, ge), targets, gl, ge, 1.0)


@pytest.mark.parametrize("type", list(TYPES))
@pytest.mark.parametrize("rows", [9, 700])
@pytest.mark.parametrize("vocab,pads,offsets", [(2048, (8, 16), (0, 0)), (2048, (1, 0), (3, 0)),
                                                (50001, (0, 0), (1, 1)), (50001, (7, 0), (5, 2)),
                                                (777, (3, 3), (2, 2)), (9001, (0, 8), (1, 3))])
def test_scoring_gradient_strides(dev, type, vocab, pads, offsets, rows):
    rows = min(rows, 9 if vocab > 4200 else rows)
    rng = np.random.default_rng(vocab)
    z = Rows(dev, logits(rng, rows, vocab), type, pads[0], offsets[0])
    targets = rng.integers(0, vocab, rows)
    gl, ge = rng.standard_normal(rows).astype(np.float32), rng.standard_normal(rows).astype(np.float32)
    out = z.like(pads[1], offsets[1])
    got = score_gradient(dev, z, targets, gl, ge, 1.7, out)
    check_score_gradient(z, got, targets, gl, ge, 1.7)
    assert out.untouched() and z.untouched()
    # in place
    got2 = score_gradient(dev, z, targets, gl, ge, 1.7, z)
    np.testing.assert_array_equal(got, got2)
    assert z.untouched()


@pytest.mark.parametrize("type", list(TYPES))
@pytest.mark.parametrize("vocab,many", [(130, False), (2048, False), (20001, False), (130, True), (2048, True)])
def test_scoring_gradient_masks(dev, type, vocab, many):
    rng = np.random.default_rng(11)
    z = logits(rng, 7, vocab)
    z[0, rng.random(vocab) < 0.5] = -np.inf
    z[1] = -np.inf
    z[2, 1:] = -np.inf
    z[3, :-2] = {"f32": -3.4028234663852886e38, "f16": -65504.0, "bf16": -3.3895313892515355e38}[type]
    z[4, 7] = np.nan
    targets = np.array([int(np.argmax(z[0])), 3, 0, vocab - 1, 0, NO, 2], np.uint32)
    gl, ge = rng.standard_normal(7).astype(np.float32), rng.standard_normal(7).astype(np.float32)
    gl[4] = ge[4] = 0  # nothing comes in: zeros, in spite of the NaN
    z, targets, gl, ge = repeat(many, z, targets, gl, ge)
    z = Rows(dev, z, type)
    got = score_gradient(dev, z, targets, gl, ge)
    assert not got[4::7].any()
    z.host[4::7] = 0
    check_score_gradient(z, got, targets, gl, ge, 1.0)
    for one in (dict(gl=gl, ge=None), dict(gl=None, ge=ge)):
        got = score_gradient(dev, z, targets, **one)
        check_score_gradient(z, got, targets, one["gl"], one["ge"], 1.0)


# ------------------------------------------------------------- distillation

def distill(dev, z, ids, teacher, name="tl_distill_rows", tau=1.0, teacher_tau=1.0, tail=False,
            targets=None, kd=1.0, ce=0.0, scale=None, out=None, stats=None):
    rows, top = np.shape(ids)
    d = base_desc(capi.TlDistillDesc, dev, z, tau)
    d.teacher_temperature, d.tail, d.top = teacher_tau, int(tail), top
    d.kd_weight, d.ce_weight = kd, ce
    held = [u32(dev, ids), f32(dev, teacher)]
    d.teacher_ids, d.teacher = held[0].data_ptr(), held[1].data_ptr()
    if targets is not None:
        held.append(u32(dev, targets))
        d.targets = held[-1].data_ptr()
    if scale is not None:
        held.append(f32(dev, scale))
        d.row_scale = held[-1].data_ptr()
    stats = dev.empty((rows, 8)) if stats is None else stats
    loss, kl = dev.empty((rows,)), dev.empty((rows,))
    d.loss, d.kl, d.stats = loss.data_ptr(), kl.data_ptr(), stats.data_ptr()
    if out is not None:
        d.dlogits, d.d_row_stride = out.ptr(), out.stride
    call(dev, name, d)
    res = {"stats": stats}
    if name != "tl_distill_backward_rows":
        res.update(loss=dev.host(loss), kl=dev.host(kl))
    if out is not None:
        res["grad"] = out.get()
    return res


def check_distill(z, got, ids, teacher, tau=1.0, teacher_tau=1.0, tail=False, targets=None, kd=1.0,
                  ce=0.0, scale=None):
    teacher = np.asarray(teacher, np.float32)
    args = dict(temperature=tau, teacher_temperature=teacher_tau, tail=tail, targets=targets, kd=kd, ce=ce)
    p, inside, rest, some = ops._slots(ids, teacher, z.shape[1], teacher_tau, tail)
    lq = ops.log_softmax(z.host, tau)
    q, size = np.exp(lq), np.where(np.isfinite(lq), np.abs(lq), 0.0)
    es = err_sum(z.shape[1])
    lp = np.where(p > 0, np.abs(np.log(np.where(p > 0, p, 1))), 0)
    e_p = 8 * U * (1 + np.abs(np.where(np.isfinite(teacher), teacher, 0) / teacher_tau).max(-1, keepdims=True))
    # the rest of the teacher's mass is off by the p's errors together; its
    # term changes by that times 1 + |log rest - log q_r|
    e_rest = (e_p[:, 0] + 140 * U) * (p.sum(-1) + rest) if tail else np.zeros(len(p))
    with np.errstate(divide="ignore"):
        q_r = np.where(inside, 0, q).sum(-1)
        lq_r = np.where(q_r > 0, np.abs(np.log(np.where(q_r > 0, q_r, 1))), 200.0)
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
        share = np.where(inside, 0, q) / np.where(q_r > 0, q_r, 1)[:, None]
        tol = abs(kd) / tau * (q * (2 * es + 8 * U * (size + 16)) + p * (e_p + 4 * U)
                               + share * (e_rest + rest * (2 * es + 8 * U * (16 + lq_r)))[:, None])
        if targets is not None and ce:
            l1 = ops.log_softmax(z.host)
            s1 = np.where(np.isfinite(l1), np.abs(l1), 0)
            tol += abs(ce) * (np.exp(l1) * (2 * es + 8 * U * (s1 + 16)) + 4 * U * (want != 0))
        if scale is not None:
            tol *= np.abs(scale)[:, None]
        near(got["grad"], want, tol + 2 * ROUND[z.type] * np.abs(want)
             + (2.0 ** -25 if z.type == "f16" else 2.0 ** -126))


def teacher_of(rng, rows, vocab, top):
    """A teacher's `top` likeliest tokens and their log probabilities."""
    z = rng.standard_normal((rows, vocab)) * 2
    ids = ops.top(z, top)
    return z, ids.astype(np.uint32), np.take_along_axis(ops.log_softmax(z), ids, 1).astype(np.float32)


def all_three(dev, z, ids, teacher, scale, **args):
    """Forward, backward from its statistics, and both in one call."""
    one = distill(dev, z, ids, teacher, **args)
    two = distill(dev, z, ids, teacher, "tl_distill_backward_rows", scale=scale, out=z.like(),
                  stats=one["stats"], **args)
    both = distill(dev, z, ids, teacher, "tl_distill_train_rows", scale=scale, out=z.like(), **args)
    for got in (one, two, both):
        check_distill(z, got, ids, teacher, scale=scale, **args)
    return one, two, both


@pytest.mark.parametrize("type", list(TYPES))
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("rows,vocab", SIZES)
def test_distillation_sizes(dev, type, tail, rows, vocab):
    rng = np.random.default_rng(rows * 31 + vocab)
    top = min(vocab, int(rng.integers(1, 129)))
    zt, ids, teacher = teacher_of(rng, rows, vocab, top)
    z = Rows(dev, 0.7 * zt + 0.5 * rng.standard_normal((rows, vocab)), type)
    targets = rng.integers(0, vocab, rows)
    scale = rng.uniform(0.2, 2, rows).astype(np.float32)
    all_three(dev, z, ids, teacher, scale, tail=tail, targets=targets, kd=0.8, ce=0.3,
              tau=2.0 if vocab % 2 else 1.0, teacher_tau=1.0)


@pytest.mark.parametrize("type", list(TYPES))
@pytest.mark.parametrize("tail,hard", [(False, False), (True, False), (False, True), (True, True)])
@pytest.mark.parametrize("tau", [0.5, 1.0, 3.0])
def test_distillation_forms(dev, type, tail, hard, tau):
    rng = np.random.default_rng(12)
    for vocab, many in ((2048, False), (30011, False), (2048, True)):
        zt, ids, teacher = teacher_of(rng, 6, vocab, 32)
        # a target in a slot, outside the slots, and none
        targets = np.array([ids[0, 5], ids[1, 0], vocab - 1, NO, 0, NO], np.uint32)
        zt, ids, teacher, targets = repeat(many, zt, ids, teacher, targets)
        z = Rows(dev, zt + rng.standard_normal(zt.shape), type)
        all_three(dev, z, ids, teacher, np.ones(len(zt), np.float32), tail=tail, tau=tau, kd=tau * tau,
                  ce=0.25 if hard else 0.0, targets=targets if hard else None)
    # teacher's raw logits and their own temperature
    raw = np.take_along_axis(zt, ids.astype(np.int64), 1)
    all_three(dev, z, ids, raw, None, tau=tau, teacher_tau=tau)


@pytest.mark.parametrize("type", list(TYPES))
@pytest.mark.parametrize("vocab,pads,offsets", [(2048, (8, 16), (0, 0)), (2048, (1, 0), (3, 0)),
                                                (50001, (0, 0), (1, 1)), (50001, (7, 0), (5, 2)),
                                                (777, (3, 3), (2, 2)), (9001, (0, 8), (1, 3)),
                                                (131075, (0, 0), (3, 3))])
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("rows", [5, 700])
def test_distillation_strides(dev, type, vocab, pads, offsets, tail, rows):
    rows = min(rows, 5 if vocab > 4200 else rows)
    rng = np.random.default_rng(vocab)
    zt, ids, teacher = teacher_of(rng, rows, vocab, 24)
    targets = rng.integers(0, vocab, rows)
    args = dict(tail=tail, targets=targets, kd=2.0, ce=0.5, tau=1.5)
    zh = zt + 0.5 * rng.standard_normal(zt.shape)
    z = Rows(dev, zh, type, pads[0], offsets[0])
    out = z.like(pads[1], offsets[1])
    both = distill(dev, z, ids, teacher, "tl_distill_train_rows", out=out, **args)
    check_distill(z, both, ids, teacher, **args)
    assert out.untouched() and z.untouched()
    out2 = z.like(pads[1], offsets[1])
    two = distill(dev, z, ids, teacher, "tl_distill_backward_rows", out=out2, stats=both["stats"], **args)
    check_distill(z, two, ids, teacher, **args)
    assert out2.untouched()
    # in place, both ways
    for name in ("tl_distill_backward_rows", "tl_distill_train_rows"):
        z = Rows(dev, zh, type, pads[0], offsets[0])
        host = z.host
        got = distill(dev, z, ids, teacher, name, out=z, stats=both["stats"].clone(), **args)
        z.host = host
        check_distill(z, got, ids, teacher, **args)
        assert z.untouched()


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("vocab,many", [(100, False), (2048, False), (40001, False), (100, True), (2048, True)])
def test_distillation_slots_and_masks(dev, tail, vocab, many):
    """Empty slots, rows without slots, values of -inf, a student that cannot
    say a slot's token, nothing outside the slots, nothing at all, a student
    whose mass outside the slots is far below fp32's range."""
    rng = np.random.default_rng(13)
    rows, top = 10, 50
    zt, ids, teacher = teacher_of(rng, rows, vocab, top)
    z = zt.copy()
    ids[0, 7:] = NO
    ids[1] = NO
    teacher[2, ::2] = -np.inf
    teacher[3] = -np.inf
    z[4, ids[4, 0]] = -np.inf                                    # KL is +inf, the gradient is not
    z[5, np.setdiff1d(np.arange(vocab), ids[5])] = -np.inf       # nothing outside the slots
    z[6] = -np.inf
    z[7, np.setdiff1d(np.arange(vocab), ids[7])] -= 300          # underflows outside the slots
    z[8, ids[8].astype(np.int64)] -= 300                         # and within
    targets = np.array([0, 1, 2, NO, 3, int(ids[5, 0]), 5, int(ids[7, 1]), 6, NO], np.uint32)
    z, ids, teacher, targets = repeat(many, z, ids, teacher, targets)
    zr = Rows(dev, z)
    one, two, both = all_three(dev, zr, ids, teacher, rng.uniform(.5, 1.5, len(z)).astype(np.float32),
                               tail=tail, targets=targets, ce=0.5)
    assert one["kl"][1] == one["kl"][3] == 0 and np.isposinf(one["kl"][[4, 6]]).all()
    assert np.isfinite(both["grad"]).all() and not both["grad"][6].any()


@pytest.mark.parametrize("rows,vocab", [(2, 50001), (5, 131072), (200, 5000), (900, 2048)])
def test_rows_at_the_lowest_value(dev, rows, vocab):
    """Rows whose every logit (outside a few) is fp32's lowest value, beyond
    what sums in powers of two hold: in a cluster, a CTA and a warp per row,
    the gradient beside the logits and in their place."""
    rng = np.random.default_rng(21)
    zh = np.full((rows, vocab), -3.4028234663852886e38)
    zh[1::2, vocab // 3] = 2.0
    ids = np.stack([rng.permutation(vocab)[:8] for _ in range(rows)]).astype(np.uint32)
    teacher = np.log(np.tile([.3, .2, .1, .1, .05, .05, .02, .01], (rows, 1)))
    targets = rng.integers(0, vocab, rows)
    # (log q of a wiped-out token is -3e38, its KL beyond fp32: gradients only)
    for tail in (False, True):
        args = dict(tail=tail, targets=targets, ce=0.5, kd=0.7)
        z = Rows(dev, zh)
        want = ops.distill_gradient(z.host, ids, np.asarray(teacher, np.float32), **args)
        grads = []
        for out in (z.like(), z):
            grads.append(distill(dev, z, ids, teacher, "tl_distill_train_rows", out=out, **args)["grad"])
        np.testing.assert_array_equal(grads[0], grads[1])
        near(grads[0], want, 1e-5 * np.abs(want) + 1e-6)
    z = Rows(dev, zh)
    check_score(z, score(dev, z, targets, 20), targets, 20, 1.0)
    one = np.ones(rows, np.float32)
    check_score_gradient(z, score_gradient(dev, z, targets, one, one), targets, one, one, 1.0)


def test_distillation_every_token_in_a_slot(dev):
    rng = np.random.default_rng(14)
    for rows in (5, 700):
        zt, ids, teacher = teacher_of(rng, rows, 64, 64)
        for tail in (False, True):
            all_three(dev, Rows(dev, rng.standard_normal((rows, 64))), ids, teacher, None, tail=tail)


def test_distillation_ids_out_of_range(dev):
    rng = np.random.default_rng(15)
    zt, ids, teacher = teacher_of(rng, 4, 500, 8)
    z = Rows(dev, zt)
    assert dev.status() == 0
    ids[2, 3] = 500
    distill(dev, z, ids, teacher)
    assert dev.status() == capi.TL_FLAG_INDEX_RANGE
    all_three(dev, z, ids, teacher, None, tail=True)
    assert dev.status() == capi.TL_FLAG_INDEX_RANGE
    ids[2, 3] = NO
    targets = np.array([0, 1, 777, NO], np.uint32)
    all_three(dev, z, ids, teacher, None, targets=targets, ce=1.0)
    assert dev.status() == capi.TL_FLAG_INDEX_RANGE


def test_distillation_rows_without_gradient(dev):
    """A scale of 0 gives zeros, whatever the logits."""
    rng = np.random.default_rng(16)
    for vocab, many in ((300, False), (2048, False), (20001, False), (2048, True)):
        zt, ids, teacher = teacher_of(rng, 3, vocab, 4)
        zt[1, 5] = np.nan
        zt, ids, teacher, scale = repeat(many, zt, ids, teacher, np.array([1, 0, 2], np.float32))
        z = Rows(dev, zt)
        got = distill(dev, z, ids, teacher, "tl_distill_train_rows", scale=scale, out=z.like())
        assert not got["grad"][1].any() and np.isnan(got["kl"][1])
        two = distill(dev, z, ids, teacher, "tl_distill_backward_rows", scale=scale, out=z.like(),
                      stats=got["stats"])
        assert not two["grad"][1].any()
        np.testing.assert_array_equal(got["grad"][[0, 2]] != 0, two["grad"][[0, 2]] != 0)


def test_distillation_repeats_bit_for_bit(dev):
    rng = np.random.default_rng(17)
    for type, rows, vocab in (("f32", 50, 2048), ("bf16", 3, 50001), ("f16", 2, 131072), ("f32", 700, 2048)):
        zt, ids, teacher = teacher_of(rng, rows, vocab, 32)
        z = Rows(dev, zt, type)
        args = dict(tail=True, targets=rng.integers(0, vocab, rows), ce=0.5, tau=2.0)
        runs = [distill(dev, z, ids, teacher, "tl_distill_train_rows", out=z.like(), **args) for _ in range(3)]
        for r in runs[1:]:
            for k in ("loss", "kl", "grad"):
                np.testing.assert_array_equal(r[k], runs[0][k])


@pytest.mark.parametrize("tail", [False, True])
def test_gradients_against_differences(dev, tail):
    """The gradient along a direction against the loss at both ends of a step
    h along it.  For N(0, 1) directions the loss's third derivative along
    them is of order 1: h^2 / 6 of it is 2e-5 at h = 1e-2; the losses are of
    order 5, rounded to 3e-7, over 2 h: 3e-5.  5e-4 is ten times both."""
    rng = np.random.default_rng(18)
    rows, vocab, h = 6, 300, 1e-2
    zt, ids, teacher = teacher_of(rng, rows, vocab, 16)
    zh = (0.8 * zt + 0.5 * rng.standard_normal(zt.shape)).astype(np.float32)
    way = rng.standard_normal(zt.shape).astype(np.float32)
    targets = rng.integers(0, vocab, rows)
    args = dict(tail=tail, targets=targets, ce=0.4, kd=0.9, tau=1.5)
    z = Rows(dev, zh)
    grad = distill(dev, z, ids, teacher, "tl_distill_train_rows", out=z.like(), **args)["grad"]
    ends = [distill(dev, Rows(dev, zh + s * h * way), ids, teacher, **args)["loss"].astype(np.float64)
            for s in (1, -1)]
    np.testing.assert_allclose((grad * way).sum(-1), (ends[0] - ends[1]) / (2 * h), atol=5e-4)
    one = np.ones(rows, np.float32)
    grad = score_gradient(dev, z, targets, one, 0.5 * one, 1.5)
    ends = [score(dev, Rows(dev, zh + s * h * way), targets, 0, 1.5) for s in (1, -1)]
    ends = [e["logprob"].astype(np.float64) + 0.5 * e["entropy"] for e in ends]
    np.testing.assert_allclose((grad * way).sum(-1), (ends[0] - ends[1]) / (2 * h), atol=5e-4)


# --------------------------------------------------------- memory and streams

def test_offsets_beyond_32_bits(dev):
    """Rows more than 2^32 elements apart."""
    torch = dev.torch
    stride = (1 << 32) + 8
    buf = torch.empty(2 * stride + 4096, dtype=torch.bfloat16, device=dev.dev)
    rng = np.random.default_rng(19)
    zh = rng.standard_normal((3, 4000))
    z = Rows.__new__(Rows)
    z.dev, z.type, z.stride, z.shape, z.offset, z.buf = dev, "bf16", stride, zh.shape, 0, buf
    z.view = torch.as_strided(buf, (3, 4000), (stride, 1))
    z.view.copy_(torch.from_numpy(zh))
    z.host = z.view.double().cpu().numpy()
    targets = np.array([5, 3999, 17])
    check_score(z, score(dev, z, targets, 40), targets, 40, 1.0)
    one = np.ones(3, np.float32)
    out = z.like(0)
    check_score_gradient(z, score_gradient(dev, z, targets, one, one, 1.0, out), targets, one, one, 1.0)
    _, ids, teacher = teacher_of(rng, 3, 4000, 20)
    got = distill(dev, z, ids, teacher, "tl_distill_train_rows", out=z, tail=True)
    check_distill(z, got, ids, teacher, tail=True)


def test_on_another_stream_and_in_a_graph(dev):
    torch = dev.torch
    rng = np.random.default_rng(20)
    zh = logits(rng, 20, 5000)
    z = Rows(dev, zh)
    targets = rng.integers(0, 5000, 20)
    want = score(dev, z, targets, 9)
    dev.torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = score(dev, z, targets, 9)
    for k in want:
        np.testing.assert_array_equal(got[k], want[k])
    # captured once, replayed on new logits
    d = base_desc(capi.TlTokenLogprobDesc, dev, z, 1.0)
    e = dev.empty((20,))
    d.entropy = e.data_ptr()
    lib, graph = dev.lib, ctypes.c_void_p()
    raw = ctypes.c_void_p(s.cuda_stream)
    capi.check(lib.tl_graph_capture_begin(raw), lib, "begin")
    rc = lib.tl_token_logprob_rows(ctypes.byref(d), raw)
    capi.check(lib.tl_graph_capture_end(raw, ctypes.byref(graph)), lib, "end")
    capi.check(rc, lib, "tl_token_logprob_rows")
    z2 = logits(rng, 20, 5000)
    with torch.cuda.stream(s):
        z.view.copy_(torch.from_numpy(z2))
    capi.check(lib.tl_graph_launch(graph, raw), lib, "launch")
    torch.cuda.synchronize()
    near(dev.host(e), ops.entropy(z2.astype(np.float32)), 1e-4)
    capi.check(lib.tl_graph_destroy(graph), lib, "destroy")
