"""Training attention with rotated heads, as a step uses it: tl_rotary_heads out of
the rows that one product wrote ([B, T, 3, H, D]), tl_flash_attention_fwd and _bwd,
tl_rotary_heads_backward into the rows' gradient, against the float64 oracle; and
the same sequences answered from a paged cache.

Tolerances: tests/test_flash_attention_gpu.py gives each TF32 product on a path 1e-3
of the result's Frobenius norm (O and dV 2, dQ and dK 3), the rotation's own rounding
is below 1e-5 of it.  The gradient dx = R^T of (g w - x^ mean(g w x^)) / rms is a
contraction of g up to max |w| / min rms, so that an error of 3e-3 ||g|| in g is at
most that many times as much in dx; a weight's gradient, the sum of g x^ over rows,
is off by at most 3e-3 ||g|| ||x^|| (Cauchy-Schwarz, over all elements together)."""
import ctypes
import math

import numpy as np
import pytest

from oracle import head_ops, ops
from templit_b200 import capi
from tests.helpers import Dev
from tests.test_rotary_gpu import table

pytestmark = pytest.mark.gpu
B, H, D = 2, 6, 64


@pytest.fixture(scope="module")
def dev():
    return Dev()


def head_view(x):
    """[B, T, H, D]"""
    s = x.stride()
    return capi.TlHeadView(x.data_ptr(), s[0], s[2], s[1])


def attn_view(x):
    v, s = capi.TlAttnView(), x.stride()
    v.p, v.batch_stride, v.head_stride, v.row_stride = x.data_ptr(), s[0], s[2], s[1]
    return v


def by_head(x):
    return np.swapaxes(x, 1, 2)


def off(got, want):
    return np.linalg.norm(np.asarray(got, np.float64) - want)


@pytest.mark.parametrize("T, rotary, norm, interleaved", [(192, 64, 0, 0), (192, 64, 1, 0), (77, 32, 1, 1)])
def test_training_step(dev, T, rotary, norm, interleaved):
    rng = np.random.default_rng(T + norm)
    t = dev.torch
    rows = dev.t(rng.standard_normal((B, T, 3, H, D)).astype(np.float32))
    d_o = dev.t(rng.standard_normal((B, T, H, D)).astype(np.float32))
    weights = [dev.t((1 + 0.3 * rng.standard_normal(D)).astype(np.float32)) for _ in range(2)]
    freq, mag, radians = table(dev, rotary)
    new = lambda *s: t.full(s, 7.0, device=dev.dev)  # noqa: E731
    q, k, o, dq, dk = (new(B, T, H, D) for _ in range(5))
    d_rows, lse, delta = new(B, T, 3, H, D), new(B, H, T), new(B, H, T)
    d_weights = [new(D) for _ in range(2)]
    mask = dev.t(ops.causal_mask(T).astype(np.float32))
    divisor = dev.t(np.array([math.sqrt(D)], np.float32))

    r = capi.TlRotaryDesc(B=B, T=T, D=D, rotary_dim=rotary, type=capi.TL_FLOAT32, out_type=capi.TL_FLOAT32,
                          layout=interleaved, norm=norm, eps=1e-6, magnitude=mag, frequencies=freq.data_ptr())
    for part, i, out, g in ((r.q, 0, q, dq), (r.k, 1, k, dk)):
        part.heads, part.x, part.out, part.d_out = H, head_view(rows[:, :, i]), head_view(out), head_view(g)
        part.dx = head_view(d_rows[:, :, i])
        if norm:
            part.weight, part.dweight = weights[i].data_ptr(), d_weights[i].data_ptr()
    ws = dev.ws(dev.lib.tl_rotary_heads_workspace_size(ctypes.byref(r)))
    r.workspace, r.workspace_bytes = ws.data_ptr(), ws.numel()
    f = capi.TlFlashDesc(B=B, T=T, H=H, D=D, divisor=divisor.data_ptr(), mask=mask.data_ptr(), lse=lse.data_ptr(),
                         delta=delta.data_ptr())
    f.q, f.k, f.v, f.o, f.d_o = (attn_view(x) for x in (q, k, rows[:, :, 2], o, d_o))
    f.dq, f.dk, f.dv = attn_view(dq), attn_view(dk), attn_view(d_rows[:, :, 2])
    assert dev.lib.tl_flash_attention_supported(ctypes.byref(f))
    for call, d in (("tl_rotary_heads", r), ("tl_flash_attention_fwd", f), ("tl_flash_attention_bwd", f),
                    ("tl_rotary_heads_backward", r)):
        capi.check(getattr(dev.lib, call)(ctypes.byref(d), dev.stream), dev.lib, call)
    t.cuda.synchronize()

    x = rows.double().cpu().numpy()
    w = [a.double().cpu().numpy() if norm else None for a in weights]
    kw = dict(interleaved=bool(interleaved), magnitude=mag, normed=bool(norm))
    turned = [head_ops.heads(x[:, :, i], np.arange(T)[None], radians, weight=w[i], **kw) for i in range(2)]
    hq, hk, hv, hg = (by_head(a) for a in (turned[0], turned[1], x[:, :, 2], d_o.double().cpu().numpy()))
    divide = math.sqrt(D)
    p, want_o = ops.attention_forward(hq, hk, hv, divide, ops.causal_mask(T))
    grads = ops.attention_backward(hq, hk, hv, p, divide, hg)
    assert off(by_head(o.cpu().numpy()), want_o) <= 2e-3 * np.linalg.norm(want_o)
    got = d_rows.cpu().numpy()
    assert off(by_head(got[:, :, 2]), grads[2]) <= 2e-3 * np.linalg.norm(grads[2])
    for i in range(2):
        g = by_head(grads[i])
        want, want_weight = head_ops.heads_gradient(x[:, :, i], g, np.arange(T)[None], radians, bool(interleaved), mag,
                                                    bool(norm), w[i])
        rms = np.sqrt((x[:, :, i] ** 2).mean(-1, keepdims=True) + 1e-6)
        grow = np.abs(w[i]).max() / rms.min() if norm else 1.0
        assert off(got[:, :, i], want) <= (3e-3 * grow + 1e-5) * np.linalg.norm(g)
        if norm:
            assert off(d_weights[i].cpu().numpy(), want_weight) <= (3e-3 + 1e-5) * np.linalg.norm(g) * np.linalg.norm(x[:, :, i] / rms)
    assert dev.status() == 0


def test_a_cache_answers_as_the_training_forward(dev):
    """Two sequences of 192 tokens, 6 heads of 64: written into pages and attended there, against the
    training kernel on the same numbers (its TF32 products: 2e-3 of the norm)."""
    T, page = 192, 16
    rng = np.random.default_rng(4)
    t = dev.torch
    rows = dev.t(rng.standard_normal((B, T, 3, H, D)).astype(np.float32))
    freq, mag, _ = table(dev, D)
    new = lambda *s: t.full(s, 7.0, device=dev.dev)  # noqa: E731
    q, k, o = (new(B, T, H, D) for _ in range(3))
    r = capi.TlRotaryDesc(B=B, T=T, D=D, rotary_dim=D, type=capi.TL_FLOAT32, out_type=capi.TL_FLOAT32, magnitude=mag,
                          frequencies=freq.data_ptr())
    for part, i, out in ((r.q, 0, q), (r.k, 1, k)):
        part.heads, part.x, part.out = H, head_view(rows[:, :, i]), head_view(out)
    lse, delta = new(B, H, T), new(B, H, T)
    mask, divisor = dev.t(ops.causal_mask(T).astype(np.float32)), dev.t(np.array([math.sqrt(D)], np.float32))
    f = capi.TlFlashDesc(B=B, T=T, H=H, D=D, divisor=divisor.data_ptr(), mask=mask.data_ptr(), lse=lse.data_ptr(),
                         delta=delta.data_ptr())
    f.q, f.k, f.v, f.o = (attn_view(x) for x in (q, k, rows[:, :, 2], o))
    capi.check(dev.lib.tl_rotary_heads(ctypes.byref(r), dev.stream), dev.lib)
    capi.check(dev.lib.tl_flash_attention_fwd(ctypes.byref(f), dev.stream), dev.lib)

    pages = B * T // page
    cache_k, cache_v = (new(pages, page, H, D) for _ in range(2))
    blocks = t.randperm(pages, device=dev.dev).to(t.int32).view(B, T // page)
    starts, lengths = dev.t(np.array([0, T, 2 * T]), np.uint32), dev.t(np.array([T, T]), np.uint32)
    tokens = rows.view(B * T, 3, H, D)
    turned, out = new(B * T, H, D), new(B * T, H, D)
    view = lambda x: capi.TlHeadView(x.data_ptr(), 0, x.stride(-2), x.stride(-3))  # noqa: E731
    a = capi.TlCacheAppendDesc(q=view(tokens[:, 0]), k=view(tokens[:, 1]), v=view(tokens[:, 2]), q_out=view(turned),
                               q_heads=H, type=capi.TL_FLOAT32, q_out_type=capi.TL_FLOAT32, rotary_dim=D, magnitude=mag,
                               frequencies=freq.data_ptr())
    b = capi.TlPagedAttentionDesc(q=view(turned), out=view(out), q_heads=H, out_type=capi.TL_FLOAT32, causal=1,
                                  scale=1 / math.sqrt(D))
    for d in (a, b):
        c = d.cache
        c.k, c.v, c.page_stride, c.slot_stride, c.head_stride = (cache_k.data_ptr(), cache_v.data_ptr(),
                                                                 *cache_k.stride()[:3])
        c.pages, c.page_size, c.heads, c.D, c.type = pages, page, H, D, capi.TL_FLOAT32
        c.table, c.starts, c.lengths = blocks.data_ptr(), starts.data_ptr(), lengths.data_ptr()
        c.sequences, c.tokens, c.table_stride = B, B * T, T // page
    ws = dev.ws(dev.lib.tl_paged_attention_workspace_size(ctypes.byref(b)))
    b.workspace, b.workspace_bytes = ws.data_ptr(), ws.numel()
    capi.check(dev.lib.tl_cache_append(ctypes.byref(a), dev.stream), dev.lib)
    capi.check(dev.lib.tl_paged_attention(ctypes.byref(b), dev.stream), dev.lib)
    t.cuda.synchronize()
    assert (turned.view(B, T, H, D) == q).all()
    want = o.double().cpu().numpy()
    assert off(out.view(B, T, H, D).cpu().numpy(), want) <= 2e-3 * np.linalg.norm(want)
    assert dev.status() == 0
