"""The oracle of rotation, head norms and cached attention (oracle/head_ops.py)
against differences and known properties, and tl_rotary_frequencies, which
runs on the host, against it."""
import ctypes

import numpy as np
import pytest

from oracle import head_ops as ops
from templit_b200 import capi

SPECS = [(ops.PLAIN, 1.0, 0.0, 0.0, 0.0), (ops.LINEAR, 4.0, 0.0, 0.0, 0.0), (ops.NTK, 8.0, 0.0, 0.0, 0.0),
         (ops.PARTS, 8.0, 4096.0, 1.0, 32.0), (ops.PARTS, 1.0, 4096.0, 1.0, 32.0), (ops.SMOOTH, 8.0, 8192.0, 1.0, 4.0)]


@pytest.mark.parametrize("dim", [2, 4, 20, 64, 128, 256])
@pytest.mark.parametrize("base", [1.5, 10000.0, 5e6])
@pytest.mark.parametrize("scaling,factor,original,low,high", SPECS)
def test_frequencies(dim, base, scaling, factor, original, low, high):
    if scaling == ops.NTK and dim == 2:
        return
    want, magnitude = ops.frequencies(dim, base, scaling, factor, original, low, high)
    spec = capi.TlRotarySpec(base=base, factor=factor, original_length=original, low=low, high=high, dim=dim,
                             scaling=scaling)
    got, mag = (ctypes.c_uint64 * (dim // 2))(), ctypes.c_float()
    lib = capi.cuda_lib()
    capi.check(lib.tl_rotary_frequencies(ctypes.byref(spec), got, ctypes.byref(mag)), lib)
    turns = np.array([int(x) for x in got], dtype=object) / 2 ** 64
    np.testing.assert_allclose(turns.astype(np.float64), want / (2 * np.pi), rtol=1e-13, atol=2.0 ** -63)
    assert mag.value == pytest.approx(magnitude, rel=2 ** -23)


def test_frequencies_refusals():
    lib = capi.cuda_lib()
    out = (ctypes.c_uint64 * 128)()
    good = dict(base=10000.0, factor=2.0, original_length=64.0, low=1.0, high=2.0, dim=64, scaling=ops.PARTS)
    assert lib.tl_rotary_frequencies(ctypes.byref(capi.TlRotarySpec(**good)), out, None) == capi.TL_OK
    for bad in (dict(base=1.0), dict(base=float("nan")), dict(base=float("inf")), dict(factor=0.5),
                dict(factor=float("nan")), dict(original_length=0.0), dict(low=0.0), dict(high=1.0), dict(scaling=5),
                dict(scaling=-1), dict(scaling=ops.NTK, dim=2)):
        assert lib.tl_rotary_frequencies(ctypes.byref(capi.TlRotarySpec(**{**good, **bad})), out, None) == capi.TL_ERR_INVALID, bad
        assert b"tl_rotary_frequencies" in lib.tl_last_error()
    for dim in (0, 1, 63, 258):
        spec = capi.TlRotarySpec(**{**good, "dim": dim})
        assert lib.tl_rotary_frequencies(ctypes.byref(spec), out, None) == capi.TL_ERR_RANGE
    assert lib.tl_rotary_frequencies(None, out, None) == capi.TL_ERR_INVALID
    assert lib.tl_rotary_frequencies(ctypes.byref(capi.TlRotarySpec(**good)), None, None) == capi.TL_ERR_INVALID


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("normed,weighted", [(False, False), (True, False), (True, True)])
def test_gradient_against_differences(interleaved, normed, weighted):
    rng = np.random.default_rng(1)
    x, g = rng.standard_normal((2, 3, 2, 10)), rng.standard_normal((2, 3, 2, 10))
    w = 1 + 0.3 * rng.standard_normal(10) if weighted else None
    at, f = rng.integers(0, 1000, (2, 3)), ops.frequencies(6)[0]
    kw = dict(interleaved=interleaved, magnitude=1.25, normed=normed, weight=w)
    dx, dw = ops.heads_gradient(x, g, at, f, **kw)
    h = 1e-6
    for _ in range(40):
        i = tuple(rng.integers(0, n) for n in x.shape)
        up, down = x.copy(), x.copy()
        up[i] += h
        down[i] -= h
        diff = ((ops.heads(up, at, f, **kw) - ops.heads(down, at, f, **kw)) * g).sum() / (2 * h)
        assert dx[i] == pytest.approx(diff, rel=1e-6, abs=1e-8)
    if weighted:
        for d in range(10):
            up, down = w.copy(), w.copy()
            up[d] += h
            down[d] -= h
            diff = ((ops.heads(x, at, f, **{**kw, "weight": up}) - ops.heads(x, at, f, **{**kw, "weight": down})) * g).sum() / (2 * h)
            assert dw[d] == pytest.approx(diff, rel=1e-6, abs=1e-8)


@pytest.mark.parametrize("interleaved", [False, True])
def test_scores_depend_on_distance_only(interleaved):
    rng = np.random.default_rng(2)
    q, k = rng.standard_normal((1, 1, 16)), rng.standard_normal((1, 1, 16))
    f = ops.frequencies(16)[0]
    at = lambda p, r: (ops.turn(q, [p], f, interleaved) * ops.turn(k, [r], f, interleaved)).sum()  # noqa: E731
    assert at(7, 3) == pytest.approx(at(1007, 1003), rel=1e-9)


def test_attention_against_whole_softmax():
    rng = np.random.default_rng(3)
    q, k, v = rng.standard_normal((4, 6, 8)), rng.standard_normal((9, 2, 8)), rng.standard_normal((9, 2, 8))
    for causal, window in ((False, 0), (True, 0), (True, 3)):
        out, lse, size = ops.attention(q, k, v, 0.3, causal, window)
        x = np.einsum("nhd,khd->nhk", q, k.repeat(3, 1)) * 0.3
        at = 5 + np.arange(4)[:, None]
        j = np.arange(9)[None]
        hide = np.zeros((4, 9), bool)
        if causal:
            hide |= j > at
        if window:
            hide |= j <= at - window
        x = np.where(hide[:, None], -np.inf, x)
        e = np.exp(x - x.max(-1, keepdims=True))
        p = e / e.sum(-1, keepdims=True)
        np.testing.assert_allclose(out, np.einsum("nhk,khd->nhd", p, v.repeat(3, 1)), rtol=1e-12, atol=1e-14)
        np.testing.assert_allclose(lse, np.log(np.exp(x).sum(-1)), rtol=1e-12)
        assert (size >= np.abs(out) - 1e-12).all()


def test_attention_rows_without_keys():
    rng = np.random.default_rng(4)
    q = rng.standard_normal((5, 2, 8))
    k, v = rng.standard_normal((3, 1, 8)), rng.standard_normal((3, 1, 8))
    out, lse, _ = ops.attention(q, k, v, 1.0)
    assert (out[:2] == 0).all() and np.isneginf(lse[:2]).all() and np.isfinite(lse[2:]).all()
