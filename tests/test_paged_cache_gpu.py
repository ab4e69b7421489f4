"""The paged cache's writer (tl_cache_append) and attention over it
(tl_paged_attention) against the float64 oracle (oracle/head_ops.py) on the
numbers as the kernels hold them.  Slots that no sequence has hold NaN.

Tolerances of attention, from the arithmetic (u = 2^-24): a score of D
products is within dS = scale (D u + P) sum |q k| of itself, P = 2^-20 for fp32
products (split in two parts of 11 bits and more), 0 for 16-bit ones; with
log2(e) it is rounded twice more, 2 u |s|.  An exponential adds 2^-21.  So a
probability is within e = 2 (dS + 2 u |s|) + 2^-20 + (L / 64 + 64) u of itself
(numerator and sum), and ROUND of the cache's type where numerators are 16-bit
numbers; the output within that of sum p |v|, and half a unit of its type.
lse is within dS + 2 u |s| + 2^-20 + (L / 64 + 64) u + 2 u |lse|."""
import ctypes
import math

import numpy as np
import pytest

from oracle import head_ops as ops
from templit_b200 import capi
from tests.helpers import Dev
from tests.test_rotary_gpu import GUARD, NORM, ROUND, TINY, TURN, TYPES, U, pair_size, table, torch_type

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return Dev()


class Cache:
    """A batch of sequences [(new tokens, keys)] in pages of a cache; `order` is its memory order."""

    def __init__(self, dev, batch, heads, D, page, type="bf16", order="pshd", seed=0, spare=3, values=1.0, extra=0,
                 gaps=False):
        rng = np.random.default_rng(seed)
        self.dev, self.batch, self.heads, self.D, self.page, self.type = dev, batch, heads, D, page, type
        self.rng = rng
        need = [-(-keys // page) for _, keys in batch]
        self.pages = sum(need) + spare
        dt = torch_type(dev, type)
        nan = float("nan")
        full = lambda *s: dev.torch.full(s, nan, dtype=dt, device=dev.dev)  # noqa: E731
        if order == "pshd":
            self.k, self.v = full(self.pages, page, heads, D), full(self.pages, page, heads, D)
        elif order == "phsd":
            self.k, self.v = (full(self.pages, heads, page, D).transpose(1, 2) for _ in range(2))
        else:  # keys and values of a page side by side, rows padded by a vector
            both = full(self.pages, 2, page, heads, D + 16)
            self.k, self.v = both[:, 0, :, :, :D], both[:, 1, :, :, :D]
        ids = rng.permutation(self.pages).astype(np.uint32)
        width = max(need + [1]) + 1
        self.table = rng.integers(0, 1 << 32, (len(batch), width), dtype=np.uint64).astype(np.uint32)  # rubbish behind the end
        used = 0
        for s, n in enumerate(need):
            self.table[s, :n] = ids[used:used + n]
            used += n
        new = [n for n, _ in batch]
        self.starts = np.concatenate(([2 if gaps else 0], np.cumsum(new) + (2 if gaps else 0))).astype(np.uint32)
        self.tokens = int(self.starts[-1]) + extra
        self.lengths = np.array([k for _, k in batch], np.uint32)
        # keys and values of every sequence
        self.keys, self.vals = [], []
        for s, (_, n) in enumerate(batch):
            k, v = rng.standard_normal((n, heads, D)), rng.standard_normal((n, heads, D)) * values
            self.keys.append(self.put(self.k, s, k))
            self.vals.append(self.put(self.v, s, v))
        self.c_table, self.c_starts, self.c_lengths = (dev.t(a, np.uint32) for a in (self.table, self.starts, self.lengths))

    def places(self, s, a=0, b=None):
        j = np.arange(a, self.batch[s][1] if b is None else b)
        t = self.dev.torch
        return t.from_numpy(self.table[s, j // self.page].astype(np.int64)).to(self.dev.dev), t.from_numpy(j % self.page).to(self.dev.dev)

    def put(self, cache, s, values):
        page, slot = self.places(s, 0, len(values))
        x = self.dev.torch.from_numpy(values).to(self.dev.dev).to(cache.dtype)
        cache[page, slot] = x
        return x.double().cpu().numpy()

    def fill(self, c):
        c.k, c.v = self.k.data_ptr(), self.v.data_ptr()
        c.page_stride, c.slot_stride, c.head_stride = self.k.stride()[:3]
        c.pages, c.page_size, c.heads, c.D, c.type = self.pages, self.page, self.heads, self.D, TYPES[self.type]
        c.table, c.starts, c.lengths = (x.data_ptr() for x in (self.c_table, self.c_starts, self.c_lengths))
        c.sequences, c.tokens, c.table_stride = len(self.batch), self.tokens, self.table.shape[1]


def view(x):
    return capi.TlHeadView(x.data_ptr(), 0, x.stride(-2), x.stride(-3))


def attend(dev, c, hq, causal=1, window=0, out_type=None, scale=None, max_length=0, max_new=0, sharp=1.0, q=None,
           stream=None, prepare_only=False):
    t = dev.torch
    if q is None:
        q = t.from_numpy(c.rng.standard_normal((c.tokens, hq, c.D)) * sharp).to(dev.dev).to(torch_type(dev, c.type))
    out = t.full((c.tokens, hq, c.D), GUARD, dtype=torch_type(dev, out_type or c.type), device=dev.dev)
    lse = t.full((c.tokens, hq), GUARD, device=dev.dev)
    d = capi.TlPagedAttentionDesc(q=view(q), out=view(out), q_heads=hq, out_type=TYPES[out_type or c.type], causal=causal,
                                  window=window, scale=scale if scale is not None else 1 / math.sqrt(c.D),
                                  lse=lse.data_ptr(), max_length=max_length, max_new=max_new)
    c.fill(d.cache)
    ws = dev.ws(dev.lib.tl_paged_attention_workspace_size(ctypes.byref(d)))
    d.workspace, d.workspace_bytes = ws.data_ptr(), dev.lib.tl_paged_attention_workspace_size(ctypes.byref(d))
    state = dict(d=d, q=q, out=out, lse=lse, ws=ws)
    if not prepare_only:
        capi.check(dev.lib.tl_paged_attention(ctypes.byref(d), stream or dev.stream), dev.lib, "tl_paged_attention")
    return state


def check(dev, c, s, causal=1, window=0):
    d, out_type = s["d"], {v: k for k, v in TYPES.items()}[s["d"].out_type]
    out, lse, q = s["out"].double().cpu().numpy(), s["lse"].double().cpu().numpy(), s["q"].double().cpu().numpy()
    seen = np.zeros(c.tokens, bool)
    for i, (new, keys) in enumerate(c.batch):
        at = slice(int(c.starts[i]), int(c.starts[i]) + new)
        seen[at] = True
        if not new:
            continue
        k, v = c.keys[i], c.vals[i]
        want, wlse, size = ops.attention(q[at], k, v, d.scale, causal, window)
        group = q.shape[1] // c.heads
        products = np.zeros(wlse.shape)
        if keys:
            norm_q = np.abs(q[at])
            with np.errstate(invalid="ignore"):
                most = np.nanmax(np.where(np.isfinite(k), np.abs(k), 0), 0).repeat(group, 0)  # [hq, D]
            products = abs(d.scale) * (norm_q * most[None]).sum(-1)
        ds = products * (c.D * U + (2.0 ** -20 if c.type == "f32" else 0)) + 2 * U * products * 1.5
        longs = 2.0 ** -20 + (keys / 64 + 64) * U
        e = 2 * ds + longs + (0 if c.type == "f32" else ROUND[c.type])
        err = size * e[..., None] + np.abs(want) * ROUND[out_type] + TINY[out_type] + 2.0 ** -126
        got = out[at]
        nan = np.isnan(want)
        assert (np.isnan(got) == nan).all(), (i, np.argwhere(np.isnan(got) != nan)[:5])
        fine = np.isfinite(want)
        with np.errstate(invalid="ignore"):
            worst = (np.abs(got - want) / err)[fine].max(initial=0)
        assert worst <= 1, (i, new, keys, worst)
        assert (got[np.isinf(want)] == want[np.isinf(want)]).all()
        none = np.isneginf(wlse)
        assert (np.isneginf(lse[at]) == none).all() and (got[none] == 0).all()
        ok = np.isfinite(wlse)
        lerr = ds + longs + 2 * U * np.abs(wlse)
        off = np.abs(lse[at][ok] - wlse[ok])
        assert (off <= lerr[ok]).all(), (i, off.max())
    # rows of no sequence are as they were
    assert (out[~seen] == GUARD).all() and (lse[~seen] == GUARD).all()
    assert dev.status() == 0


BATCHES = {
    "one": [(1, 1)],
    "one_token": [(1, 192)],
    "steps": [(1, 5), (1, 64), (1, 65), (1, 300), (1, 1), (1, 129)],
    "chunks": [(3, 3), (17, 40), (1, 90), (0, 30), (64, 64), (33, 200)],
    "empty": [(0, 0), (2, 2), (0, 0), (0, 5)],
    "more_new_than_keys": [(5, 3), (4, 0), (1, 0), (2, 2)],
}


@pytest.mark.parametrize("batch", BATCHES)
@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hq,hk,D,page", [(6, 6, 64, 16), (8, 2, 128, 16), (7, 1, 64, 5), (6, 2, 80, 1), (3, 3, 8, 33),
                                          (40, 2, 128, 64), (4, 4, 40, 7)])
def test_attention(dev, batch, type, hq, hk, D, page):
    c = Cache(dev, BATCHES[batch], hk, D, page, type)
    check(dev, c, attend(dev, c, hq, sharp=2.0))


@pytest.mark.parametrize("type", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("causal,window", [(0, 0), (1, 1), (1, 2), (1, 17), (1, 64), (1, 100), (1, 1000)])
@pytest.mark.parametrize("batch", ["steps", "chunks", "more_new_than_keys"])
def test_masks(dev, type, causal, window, batch):
    c = Cache(dev, BATCHES[batch], 2, 64, 16, type)
    check(dev, c, attend(dev, c, 6, causal, window), causal, window)


@pytest.mark.parametrize("order", ["pshd", "phsd", "interleaved"])
@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("batch", ["steps", "chunks"])
def test_cache_orders(dev, order, type, batch):
    c = Cache(dev, BATCHES[batch], 2, 64, 16, type, order)
    check(dev, c, attend(dev, c, 4))


@pytest.mark.parametrize("type", ["f16", "bf16"])
@pytest.mark.parametrize("batch", ["steps", "chunks"])
def test_wide_output(dev, type, batch):
    c = Cache(dev, BATCHES[batch], 2, 128, 16, type)
    check(dev, c, attend(dev, c, 8, out_type="f32"))


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("hq,hk,D", [(8, 8, 64), (8, 1, 128), (32, 8, 128)])
def test_long_caches(dev, type, hq, hk, D):
    """A few sequences of thousands of keys: their keys are shared out."""
    c = Cache(dev, [(1, 5003), (1, 3), (2, 2049), (1, 1024), (20, 4097)], hk, D, 16, type)
    check(dev, c, attend(dev, c, hq, sharp=3.0))


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hq,hk,D,batch", [(4, 2, 128, [(700, 700), (257, 1000), (1, 999), (128, 128), (129, 513)]),
                                           (7, 1, 64, [(300, 301), (37, 1500)]), (2, 2, 96, [(513, 600)])])
def test_long_chunks(dev, type, hq, hk, D, batch):
    c = Cache(dev, batch, hk, D, 16, type)
    check(dev, c, attend(dev, c, hq, sharp=2.0))


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("hq,hk,D,page", [(160, 1, 64, 16), (300, 2, 64, 24), (96, 3, 40, 8), (256, 2, 128, 32), (10, 10, 16, 40)])
def test_many_heads_a_key_head(dev, type, hq, hk, D, page):
    c = Cache(dev, [(3, 70), (1, 1), (17, 200)], hk, D, page, type)
    check(dev, c, attend(dev, c, hq))


@pytest.mark.parametrize("type", ["f32", "bf16"])
def test_many_sequences(dev, type):
    """More sequences than threads of a CTA, most of them short or empty, with and without hints."""
    rng = np.random.default_rng(11)
    batch = [(int(n), int(n + k)) for n, k in zip(rng.integers(0, 4, 1100), rng.integers(0, 40, 1100))]
    batch[700] = (30, 900)
    c = Cache(dev, batch, 1, 8, 8, type)
    for kw in ({}, dict(max_length=900, max_new=30), dict(max_length=900, max_new=4)):
        check(dev, c, attend(dev, c, 2, **kw))


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("new", [1, 40])
def test_a_cache_without_pages(dev, type, new):
    """No page at all: no key is there, whatever the table says."""
    c = Cache(dev, [(new, 50)], 2, 64, 16, type)
    s = attend(dev, c, 4, prepare_only=True)
    s["d"].cache.pages, s["d"].cache.k, s["d"].cache.v = 0, None, None
    capi.check(dev.lib.tl_paged_attention(ctypes.byref(s["d"]), dev.stream), dev.lib)
    dev.torch.cuda.synchronize()
    assert (s["out"] == 0).all() and dev.torch.isneginf(s["lse"]).all()
    assert dev.status() == capi.TL_FLAG_INDEX_RANGE


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("new", [3, 200])
def test_values_not_finite_that_all_rows_see(dev, type, new):
    c = Cache(dev, [(new, 3000)], 1, 64, 16, type)
    page, slot = c.places(0, 5, 6)
    c.v[page, slot] = float("nan")
    c.vals[0][5] = float("nan")
    s = attend(dev, c, 4)
    dev.torch.cuda.synchronize()
    assert dev.torch.isnan(s["out"].float()).all() and dev.torch.isfinite(s["lse"]).all()


@pytest.mark.parametrize("type", ["f16", "bf16"])
def test_window_in_long_chunks(dev, type):
    for window in (1, 100, 128, 129, 500):
        c = Cache(dev, [(600, 900), (3, 1200)], 2, 64, 16, type)
        check(dev, c, attend(dev, c, 4, 1, window), 1, window)


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
def test_rows_of_no_sequence(dev, type):
    c = Cache(dev, BATCHES["chunks"], 2, 64, 16, type, extra=9, gaps=True)
    check(dev, c, attend(dev, c, 4))


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("new", [6, 200])
def test_nothing_unseen_reaches_a_row(dev, type, new):
    """NaN and infinities in the keys and values of later tokens, and outside the window."""
    for window in (0, 20):
        c = Cache(dev, [(new, new + 50), (1, 70)], 2, 64, 16, type)
        for where, bad in ((new + 40, float("nan")), (new + 30, float("inf")), (3, float("-inf")), (5, float("nan"))):
            if where < 20 and not window:
                continue
            page, slot = c.places(0, where, where + 1)
            for cache, kept in ((c.k, c.keys), (c.v, c.vals)):
                cache[page, slot] = bad
                kept[0][where] = bad
        s = attend(dev, c, 4, 1, window)
        out = s["out"].float().cpu().numpy()
        clean = range(window + 6, new - 21) if window else range(0, new - 21)
        assert np.isfinite(out[list(clean)]).all()
        d, q = s["d"], s["q"].double().cpu().numpy()
        want, wlse, size = ops.attention(q[:new], c.keys[0], c.vals[0], d.scale, True, window)
        assert (np.isnan(out[:new]) == np.isnan(want)).all()
        ok = np.isfinite(want)
        assert (np.abs(out[:new] - want)[ok] <= (size * (2 * ROUND[type] + 1e-4) + 1e-6)[ok]).all()


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("batch", [[(1, 500), (2, 65)], [(150, 500)]])
def test_scores_far_apart(dev, type, batch):
    """Sharp queries (one key takes all), equal scores, and scores of the size of 1e4."""
    for sharp, scale in ((30.0, None), (0.0, None), (60.0, 1.0), (1.0, -0.3)):
        c = Cache(dev, batch, 2, 64, 16, type)
        check(dev, c, attend(dev, c, 4, sharp=sharp, scale=scale))


@pytest.mark.parametrize("type", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("new", [1, 140])
def test_many_small_probabilities(dev, type, new):
    """One key 12 above thousands of others that carry much of the sum together."""
    c = Cache(dev, [(new, 6000)], 1, 64, 16, type)
    k = np.zeros((6000, 1, 64))
    k[7, 0, 0] = 12.0
    c.keys[0] = c.put(c.k, 0, k)
    q = dev.torch.zeros(new, 2, 64, dtype=torch_type(dev, type), device=dev.dev)
    q[:, :, 0] = 1.0
    check(dev, c, attend(dev, c, 2, scale=1.0, q=q))


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("new", [1, 4, 200])
def test_scores_of_minus_infinity(dev, type, new):
    """A key whose score is -inf has no weight; a row of nothing else is 0."""
    c = Cache(dev, [(new, 300), (new, new)], 1, 64, 16, type)
    k = c.keys[0].copy()
    k[10, 0, :] = -3e38
    c.keys[0] = c.put(c.k, 0, k)
    k = np.full((new, 1, 64), -3e38)
    c.keys[1] = c.put(c.k, 1, k)
    q = dev.torch.full((2 * new, 2, 64), 100.0, dtype=torch_type(dev, type), device=dev.dev)
    s = attend(dev, c, 2, scale=1.0, q=q)
    out, lse = s["out"].double().cpu().numpy(), s["lse"].double().cpu().numpy()
    assert (out[new:] == 0).all() and np.isneginf(lse[new:]).all()
    assert np.isfinite(out[:new]).all() and np.isfinite(lse[:new]).all()
    assert dev.status() == 0


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("hint", [0, 1, 500, 10000])
def test_hints_change_nothing(dev, type, hint):
    c = Cache(dev, [(1, 500), (40, 300), (1, 2)], 2, 64, 16, type)
    s = attend(dev, c, 8, max_length=500, max_new=hint)
    check(dev, c, s)


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("new", [1, 90])
def test_bad_pages_and_lengths(dev, type, new):
    """Page ids out of range, lengths behind the table, rows out of the tensors: nothing is read or written there,
    the flag is raised, and the other sequences are right."""
    for what in ("page", "length", "max_length", "rows", "backwards"):
        c = Cache(dev, [(new, 200), (new, 100), (new, 150)], 2, 64, 16, type)
        max_length = 0
        if what == "page":
            c.c_table[1, 2] = c.pages
            c.c_table[1, 3] = 0x7fffffff
        elif what == "length":
            c.c_lengths[1] = 0x7fffff00
            # the rubbish behind its end may be anything, also a page of another sequence
        elif what == "max_length":
            max_length = 200
            c.c_lengths[1] = 201
        elif what == "rows":
            c.c_starts[3] = c.tokens + 5
        else:
            c.c_starts[1] = 3 * new + 1 if what == "backwards" else 0
        s = attend(dev, c, 4, max_length=max_length)
        dev.torch.cuda.synchronize()
        assert dev.status() == capi.TL_FLAG_INDEX_RANGE, what
        for i in (0, 1, 2):
            if (i == 1 and what != "rows") or (what == "rows" and i == 2) or (what == "backwards"):
                continue
            at = slice(i * new, (i + 1) * new)
            want, _, size = ops.attention(s["q"].double().cpu().numpy()[at], c.keys[i], c.vals[i], s["d"].scale)
            assert (np.abs(s["out"].double().cpu().numpy()[at] - want) <= size * 2 * ROUND[type] + 2e-4).all(), what
        if what == "page":  # the keys of good pages are still there
            at = slice(new, 2 * new)
            keep = np.r_[0:32, 64:100]
            if new == 1:
                want, _, size = ops.attention(s["q"].double().cpu().numpy()[at], c.keys[1][keep], c.vals[1][keep],
                                              s["d"].scale, causal=False)
                assert (np.abs(s["out"].double().cpu().numpy()[at] - want) <= size * 2 * ROUND[type] + 2e-4).all()
        if what == "rows":
            assert (s["out"][2 * new:] == GUARD).all()


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("batch", [[(1, 70), (2, 5)], [(140, 200), (3, 64)]])
@pytest.mark.parametrize("how", ["heads", "tokens", "both", "overlapping"])
def test_broadcast_queries(dev, type, batch, how):
    c = Cache(dev, batch, 2, 64, 16, type, seed=3)
    shape = (1 if how in ("tokens", "both") else c.tokens, 1 if how in ("heads", "both") else 8, 64)
    t = dev.torch
    if how == "overlapping":  # a head starts 8 elements behind the one before, a token 16
        q = t.from_numpy(c.rng.standard_normal(16 * c.tokens + 128)).to(dev.dev).to(torch_type(dev, type))
        q = q.as_strided((c.tokens, 8, 64), (16, 8, 1))
    else:
        q = t.from_numpy(c.rng.standard_normal(shape)).to(dev.dev).to(torch_type(dev, type)).expand(c.tokens, 8, 64)
    check(dev, c, attend(dev, c, 8, q=q))


@pytest.mark.parametrize("type", ["f32", "bf16"])
def test_two_streams_at_once(dev, type):
    torch = dev.torch
    cs = [Cache(dev, [(1, 3000), (1, 900)], 2, 64, 16, type, seed=1), Cache(dev, [(140, 700)], 2, 64, 16, type, seed=2)]
    states = [attend(dev, c, 8, prepare_only=True) for c in cs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cs]
    for _ in range(10):
        for s, st in zip(states, streams):
            capi.check(dev.lib.tl_paged_attention(ctypes.byref(s["d"]), ctypes.c_void_p(st.cuda_stream)), dev.lib)
    torch.cuda.synchronize()
    for c, s in zip(cs, states):
        check(dev, c, s)


@pytest.mark.parametrize("type", ["f32", "bf16"])
def test_captured_call_follows_the_lengths(dev, type):
    """A decoding step captured once and replayed as the sequences grow; the same answer as a plain call's."""
    torch = dev.torch
    full = [(1, 700), (1, 130)]
    c = Cache(dev, full, 2, 64, 16, type)
    s = attend(dev, c, 4, prepare_only=True)
    st = torch.cuda.Stream()
    stream, graph = ctypes.c_void_p(st.cuda_stream), ctypes.c_void_p()
    torch.cuda.synchronize()
    capi.check(dev.lib.tl_graph_capture_begin(stream), dev.lib)
    capi.check(dev.lib.tl_paged_attention(ctypes.byref(s["d"]), stream), dev.lib)
    capi.check(dev.lib.tl_graph_capture_end(stream, ctypes.byref(graph)), dev.lib)
    keys, vals = c.keys, c.vals
    for a, b in ((1, 1), (20, 130), (640, 64), (700, 65)):
        c.c_lengths.copy_(torch.tensor([a, b], dtype=torch.int64).to(torch.int32).view(c.c_lengths.dtype))
        torch.cuda.synchronize()
        capi.check(dev.lib.tl_graph_launch(graph, stream), dev.lib)
        torch.cuda.synchronize()
        c.batch, c.keys, c.vals = [(1, a), (1, b)], [keys[0][:a], keys[1][:b]], [vals[0][:a], vals[1][:b]]
        check(dev, c, s)
        graph_out = s["out"].clone()
        capi.check(dev.lib.tl_paged_attention(ctypes.byref(s["d"]), dev.stream), dev.lib)
        torch.cuda.synchronize()
        assert (graph_out == s["out"]).all()
    capi.check(dev.lib.tl_graph_destroy(graph), dev.lib)


def test_offsets_behind_32_bits(dev):
    """Pages farther than 2^32 elements from the cache's start."""
    torch = dev.torch
    pages, page, h, D = 3, 16, 1, 64
    stride = 1 << 32
    big = torch.empty(2 * stride + page * h * D + 64, dtype=torch.bfloat16, device=dev.dev)
    c = Cache(dev, [(1, 40), (20, 40)], h, D, page, "bf16")
    k = big.as_strided((pages, page, h, D), (stride, D, D, 1))
    v = k  # keys and values the same numbers
    tab = torch.tensor([[2, 0, 1], [1, 2, 0]], dtype=torch.int32, device=dev.dev)
    for i, p in enumerate((2, 0, 1)):
        n = 16 if i < 2 else 8
        k[p, :n] = torch.from_numpy(c.keys[0][i * 16:i * 16 + n]).to(dev.dev).to(torch.bfloat16)
    rows = [np.concatenate([k[p].double().cpu().numpy() for p in order])[:40] for order in ((2, 0, 1), (1, 2, 0))]
    c.k, c.v, c.pages = k, v, pages
    k[1, 8:] = 0
    rows = [np.concatenate([k[p].double().cpu().numpy() for p in order])[:40] for order in ((2, 0, 1), (1, 2, 0))]
    c.keys = c.vals = rows
    c.table, c.c_table = np.zeros((2, 3)), tab
    check(dev, c, attend(dev, c, 2))
    # and the writer
    rng = np.random.default_rng(5)
    x = torch.from_numpy(rng.standard_normal((21, 2 * h, D))).to(dev.dev).to(torch.bfloat16)
    d = capi.TlCacheAppendDesc(k=view(x[:, :h]), v=view(x[:, :h]), type=TYPES["bf16"])
    c.fill(d.cache)
    c.c_lengths.copy_(torch.tensor([40, 40]).to(torch.int32).view(c.c_lengths.dtype))
    capi.check(dev.lib.tl_cache_append(ctypes.byref(d), dev.stream), dev.lib)
    torch.cuda.synchronize()
    # sequence 1's last 20 keys are positions 20..39 of pages (1, 2, 0)
    got = torch.cat((k[2], k[0]))[4:24]
    assert (got == x[1:, :h]).all()


# ------------------------------------------------------------------- writer

def append(dev, c, hq, rotary, type, q_out_type=None, interleaved=False, norm=False, pad=0, seed=3, queries=True):
    rng = np.random.default_rng(seed)
    t, h, D = dev.torch, c.heads, c.D
    dt = torch_type(dev, type)
    row = t.from_numpy(rng.standard_normal((c.tokens, hq + 2 * h, D + pad))).to(dev.dev).to(dt)[..., :D]
    q, k, v = row[:, :hq], row[:, hq:hq + h], row[:, hq + h:]
    q_out = t.full((c.tokens, hq, D), GUARD, dtype=torch_type(dev, q_out_type or c.type), device=dev.dev)
    freq, mag, radians = table(dev, rotary) if rotary else (None, 1.0, np.zeros(0))
    qw, kw = (dev.t(1 + 0.3 * rng.standard_normal(D)) for _ in range(2)) if norm else (None, None)
    d = capi.TlCacheAppendDesc(q=view(q), k=view(k), v=view(v), q_out=view(q_out), q_heads=hq if queries else 0,
                               type=TYPES[type], q_out_type=TYPES[q_out_type or c.type], rotary_dim=rotary,
                               layout=int(interleaved), norm=int(norm), eps=1e-6, magnitude=mag,
                               frequencies=freq.data_ptr() if rotary else None, q_weight=dev.p(qw), k_weight=dev.p(kw))
    c.fill(d.cache)
    capi.check(dev.lib.tl_cache_append(ctypes.byref(d), dev.stream), dev.lib, "tl_cache_append")
    host = lambda x: x.double().cpu().numpy()  # noqa: E731
    return dict(q=host(q), k=host(k), v=host(v), q_out=q_out, radians=radians, mag=mag, norm=norm, interleaved=interleaved,
                qw=None if qw is None else host(qw), kw=None if kw is None else host(kw), q_out_type=q_out_type or c.type,
                hold=(row, freq, qw, kw), d=d)


def check_append(dev, c, s, before_k, before_v, queries=True, skip=()):
    want_k, want_v = before_k.double().cpu().numpy(), before_v.double().cpu().numpy()
    err_k = np.zeros_like(want_k)
    q_out = s["q_out"].double().cpu().numpy()
    seen = np.zeros(c.tokens, bool)

    def turned(x, at, w, type):
        y = ops.norm(x, w) if s["norm"] else x
        want = ops.turn(y, at, s["radians"], s["interleaved"], s["mag"])
        return want, pair_size(y, len(s["radians"]), s["interleaved"], s["mag"]) * (NORM if s["norm"] else TURN) + \
            np.abs(want) * 1.01 * ROUND[type] + TINY[type]

    for i, (new, keys) in enumerate(c.batch):
        if i in skip or not new:
            continue
        a = int(c.starts[i])
        seen[a:a + new] = True
        at = np.arange(keys - new, keys)
        page, slot = c.table[i, at // c.page], at % c.page
        want_k[page, slot], err_k[page, slot] = turned(s["k"][a:a + new], at, s["kw"], c.type)
        t = dev.torch
        want_v[page, slot] = t.from_numpy(s["v"][a:a + new]).to(torch_type(dev, c.type)).double().numpy()
        if queries:
            want, err = turned(s["q"][a:a + new], at, s["qw"], s["q_out_type"])
            assert (np.abs(q_out[a:a + new] - want) <= err).all()
    got_k, got_v = c.k.double().cpu().numpy(), c.v.double().cpu().numpy()
    np.testing.assert_array_equal(got_v, want_v)
    same = np.isnan(want_k)
    assert (np.isnan(got_k) == same).all()
    assert (np.abs(got_k - want_k) <= err_k)[~same].all()
    assert (q_out[~seen] == GUARD).all()


@pytest.mark.parametrize("type,cache_type,q_out_type", [("f32", "f32", None), ("bf16", "bf16", None), ("f16", "f16", None),
                                                        ("f32", "bf16", None), ("f32", "f16", "f32"), ("bf16", "f32", "bf16"),
                                                        ("f16", "f32", None)])
@pytest.mark.parametrize("D,rotary,interleaved", [(64, 64, False), (128, 64, True), (80, 0, False), (13, 6, False), (256, 256, True)])
@pytest.mark.parametrize("norm", [False, True])
def test_append(dev, type, cache_type, q_out_type, D, rotary, interleaved, norm):
    batch = [(3, 3), (1, 40), (0, 7), (20, 33), (0, 0), (1, 1)]
    for page, order in ((16, "pshd"), (5, "phsd"), (1, "interleaved")):
        c = Cache(dev, batch, 2, D, page, cache_type, order, extra=3, gaps=True)
        k, v = c.k.clone(), c.v.clone()
        s = append(dev, c, 5, rotary, type, q_out_type, interleaved, norm)
        check_append(dev, c, s, k, v)
        assert dev.status() == 0


def test_append_without_queries_and_padded_rows(dev):
    for pad in (0, 8, 3):
        c = Cache(dev, [(70, 100), (1, 2000)], 3, 64, 16, "bf16")
        k, v = c.k.clone(), c.v.clone()
        s = append(dev, c, 4, 64, "bf16", pad=pad, queries=False)
        check_append(dev, c, s, k, v, queries=False)
        assert (s["q_out"] == GUARD).all()


@pytest.mark.parametrize("sequences", [1, 31, 32, 33, 200, 1025])
def test_append_many_sequences(dev, sequences):
    rng = np.random.default_rng(sequences)
    batch = [(int(n), int(n + rng.integers(0, 9))) for n in rng.integers(0, 4, sequences)]
    c = Cache(dev, batch, 1, 8, 4, "f32")
    k, v = c.k.clone(), c.v.clone()
    check_append(dev, c, append(dev, c, 1, 8, "f32"), k, v)
    check(dev, c := Cache(dev, batch, 1, 8, 4, "f32"), attend(dev, c, 2))


def test_append_bad_places(dev):
    """Tokens without a place are not written and raise the flag; the others are written."""
    for what in ("page", "length", "short", "rows"):
        c = Cache(dev, [(2, 40), (3, 40), (2, 50)], 2, 64, 16, "bf16")
        k, v = c.k.clone(), c.v.clone()
        if what == "page":
            c.c_table[1, 2] = c.pages
        elif what == "length":
            c.c_lengths[1] = 0x70000000
        elif what == "short":
            c.c_lengths[1] = 2
        else:
            c.c_starts[3] = c.tokens + 1
        s = append(dev, c, 2, 64, "bf16")
        dev.torch.cuda.synchronize()
        assert dev.status() == capi.TL_FLAG_INDEX_RANGE, what
        check_append(dev, c, s, k, v, skip=(2,) if what == "rows" else (1,))


# ------------------------------------------------------------------ together

@pytest.mark.parametrize("type", ["f32", "bf16"])
def test_prompt_then_steps_is_the_whole_sequence(dev, type):
    """A prompt in two chunks, then single tokens, against the same tokens at once: rotation by tl_rotary_heads,
    attention over all of it."""
    rng = np.random.default_rng(9)
    t, hq, hk, D, total = dev.torch, 6, 2, 64, 150
    dt = torch_type(dev, type)
    x = t.from_numpy(rng.standard_normal((total, hq + 2 * hk, D))).to(dev.dev).to(dt)
    freq, mag, radians = table(dev, D)
    pages = t.randperm(12, device=dev.dev).to(t.int32)[None]
    caches = [t.full((12, 16, hk, D), float("nan"), dtype=dt, device=dev.dev) for _ in range(2)]
    lengths, starts = t.zeros(1, dtype=t.int32, device=dev.dev), t.zeros(2, dtype=t.int32, device=dev.dev)
    outs, done = [], 0
    for n in [100, 37] + [1] * 13:
        lengths[0], starts[1] = done + n, n
        row = x[done:done + n]
        q_out, out = t.empty(n, hq, D, dtype=dt, device=dev.dev), t.empty(n, hq, D, dtype=dt, device=dev.dev)
        a = capi.TlCacheAppendDesc(q=view(row[:, :hq]), k=view(row[:, hq:hq + hk]), v=view(row[:, hq + hk:]),
                                   q_out=view(q_out), q_heads=hq, type=TYPES[type], q_out_type=TYPES[type], rotary_dim=D,
                                   magnitude=mag, norm=1, eps=1e-6, frequencies=freq.data_ptr())
        b = capi.TlPagedAttentionDesc(q=view(q_out), out=view(out), q_heads=hq, out_type=TYPES[type], causal=1,
                                      scale=1 / math.sqrt(D))
        for d in (a, b):
            c = d.cache
            c.k, c.v, c.pages, c.page_size, c.heads, c.D, c.type = caches[0].data_ptr(), caches[1].data_ptr(), 12, 16, hk, D, TYPES[type]
            c.sequences, c.tokens, c.table_stride = 1, n, 12
            c.table, c.lengths, c.starts = pages.data_ptr(), lengths.data_ptr(), starts.data_ptr()
        ws = dev.ws(dev.lib.tl_paged_attention_workspace_size(ctypes.byref(b)))
        b.workspace, b.workspace_bytes = ws.data_ptr(), ws.numel()
        capi.check(dev.lib.tl_cache_append(ctypes.byref(a), dev.stream), dev.lib)
        capi.check(dev.lib.tl_paged_attention(ctypes.byref(b), dev.stream), dev.lib)
        outs.append(out)
        t.cuda.synchronize()
        done += n
    both = t.empty(1, total, hq + hk, D, dtype=dt, device=dev.dev)
    d = capi.TlRotaryDesc(B=1, T=total, D=D, rotary_dim=D, type=TYPES[type], out_type=TYPES[type], norm=1, eps=1e-6,
                          magnitude=mag, frequencies=freq.data_ptr())
    for part, a, b in ((d.q, 0, hq), (d.k, hq, hq + hk)):
        part.heads, part.x, part.out = b - a, view(x[:, a:b]), view(both[0, :, a:b])
    capi.check(dev.lib.tl_rotary_heads(ctypes.byref(d), dev.stream), dev.lib)
    host = both[0].double().cpu().numpy()
    # the cache holds what tl_rotary_heads gives, to the bit
    flat = caches[0][pages[0].long()].reshape(-1, hk, D)[:total]
    assert (flat == both[0, :, hq:]).all()
    want, _, size = ops.attention(host[:, :hq], host[:, hq:], x[:, hq + hk:].double().cpu().numpy(), 1 / math.sqrt(D))
    got = t.cat(outs).double().cpu().numpy()
    assert (np.abs(got - want) <= size * (ROUND[type] * 2 + 2.0 ** -17)).all()
    assert dev.status() == 0
