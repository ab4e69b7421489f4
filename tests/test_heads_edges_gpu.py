"""Edges of the rotation, cache and paged attention kernels against the
float64 oracle (oracle/head_ops.py): NaN in what a row sees, heads that do not
fill a warp without an eps, sequences that are cut, rows of one 16-bit type in
a cache of the other.  Tolerances as in test_paged_cache_gpu.py and
test_rotary_gpu.py."""
import ctypes
import math

import numpy as np
import pytest

from oracle import head_ops as ops
from templit_b200 import capi
from tests.helpers import Dev
from tests.test_paged_cache_gpu import Cache, append, attend, check, check_append
from tests.test_rotary_gpu import GUARD, NORM, ROUND, TINY, TYPES, U, Case, pair_size, torch_type

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return Dev()


# ------------------------------------------------------- NaN that a row sees

@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("batch", [[(1, 1), (1, 60)], [(1, 5003), (2, 900)], [(40, 90), (1, 3)], [(40, 5003), (20, 20)]],
                         ids=["steps", "cut_steps", "chunks", "cut_chunks"])
def test_nan_queries(dev, type, batch):
    """One NaN in a query makes all of that row's scores NaN, and its result, not the row of a token without keys."""
    c = Cache(dev, batch, 2, 64, 16, type)
    q = dev.torch.from_numpy(c.rng.standard_normal((c.tokens, 6, 64))).to(dev.dev).to(torch_type(dev, type))
    q[0, 1, 5] = float("nan")
    q[-1, 4, 63] = float("nan")
    s = attend(dev, c, 6, q=q)
    check(dev, c, s)
    lse = s["lse"].cpu().numpy()
    assert np.isnan(lse[0, 1]) and np.isnan(lse[-1, 4]) and np.isnan(lse).sum() == 2


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("new,keys,bad", [(1, 1, 0), (1, 9, 8), (1, 17, 16), (2, 65, 63), (1, 65, 64), (1, 5003, 5002), (1, 4500, 2100),
                                          (40, 40, 0), (40, 129, 128), (40, 5003, 5002), (40, 5003, 100)])
def test_a_nan_key(dev, type, new, keys, bad):
    """A NaN key reaches every row that sees it, alone in its warp's keys or not."""
    c = Cache(dev, [(new, keys)], 1, 64, 16, type)
    page, slot = c.places(0, bad, bad + 1)
    c.k[page, slot] = float("nan")
    c.keys[0][bad] = float("nan")
    s = attend(dev, c, 3)
    check(dev, c, s)
    sees = np.arange(keys - new, keys) >= bad
    assert (np.isnan(s["lse"].cpu().numpy()) == sees[:, None]).all()


# --------------------------------- values that are not finite, of later tokens

@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("out_type", [None, "f32"])
@pytest.mark.parametrize("window", [0, 50])
def test_unseen_values_in_many_sequences(dev, type, out_type, window):
    """Several pieces a CTA, cut and whole, with rows that do not see a value that is not finite."""
    rng = np.random.default_rng(4)
    batch = [(int(n), int(n + k)) for n, k in zip(rng.integers(20, 90, 160), rng.integers(0, 900, 160))]
    batch[3] = (50, 30000)
    c = Cache(dev, batch, 2, 64, 16, type)
    for i, (new, keys) in enumerate(batch):
        for bad, back in ((np.nan, 1), (np.inf, 7), (-np.inf, new), (np.nan, new + 60)):
            if rng.random() < 0.5 and 0 <= keys - back:
                page, slot = c.places(i, keys - back, keys - back + 1)
                c.v[page, slot, :, 5 + back % 40] = float(bad)
                c.vals[i][keys - back, :, 5 + back % 40] = bad
    check(dev, c, attend(dev, c, 4, 1, window, out_type), 1, window)


@pytest.mark.parametrize("type", ["f16", "bf16"])
def test_unseen_values_in_long_caches(dev, type):
    """Hundreds of thousands of keys a row, of rows that all have to be worked out again: nothing gives up."""
    t, n, new, keys, D = dev.torch, 300, 40, 200003, 64
    c = Cache(dev, [(new, keys)], 1, D, 64, type)
    page, slot = c.places(0, keys - 1, keys)
    c.v[page, slot] = float("inf")
    c.vals[0][keys - 1] = np.inf
    # every sequence reads the same pages
    c.table, c.tokens, c.batch = np.repeat(c.table, n, 0), n * new, [(new, keys)] * n
    c.c_table, c.c_starts, c.c_lengths = (dev.t(x, np.uint32) for x in (c.table, np.arange(n + 1) * new, np.full(n, keys)))
    q = t.from_numpy(c.rng.standard_normal((new, 1, D))).to(dev.dev).to(torch_type(dev, type)).repeat(n, 1, 1)
    s = attend(dev, c, 1, q=q)
    got, lse = (s[x].double().cpu().numpy().reshape(n, new, -1) for x in ("out", "lse"))
    assert dev.status() == 0
    q = q[:new].double().cpu().numpy()
    want, wlse, size = ops.attention(q, c.keys[0], c.vals[0], s["d"].scale)
    products = s["d"].scale * (np.abs(q) * np.abs(c.keys[0]).max(0)).sum(-1)
    ds, longs = products * (D * U + 3 * U), 2.0 ** -20 + (keys / 64 + 64) * U
    with np.errstate(invalid="ignore"):
        err = (size * (2 * ds + longs + ROUND[type])[..., None] + np.abs(want) * ROUND[type] + TINY[type])[:, 0]
        worst = (np.abs(got - want[:, 0]) / err)[:, :-1]
    assert worst.max() <= 1, worst.max()
    assert (got[:, -1] == np.inf).all()
    assert (np.abs(lse - wlse) <= ds + longs + 2 * U * np.abs(wlse)).all()


# ---------------------------------------------- the norm's gradient without eps

@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads", [(3, 1), (6, 6), (13, 5)])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("offset", [0, 1])  # vectors, single elements
@pytest.mark.parametrize("T", [5, 1500])
def test_norm_gradient_without_eps(dev, type, heads, D, offset, T):
    """Heads that a warp's last batch lacks add nothing to the weights' gradients, with eps = 0 too."""
    c = Case(dev, 2, T, *heads, D, D, type, norm=True, offset=offset)
    c.d.eps = 0.0
    ws = dev.ws(dev.lib.tl_rotary_heads_workspace_size(ctypes.byref(c.d)))
    c.d.workspace, c.d.workspace_bytes = ws.data_ptr(), ws.numel()
    dxs = []
    for part, x, *_ in c.parts:
        dxs.append(x.like())
        part.dx = dxs[-1].c()
    capi.check(dev.lib.tl_rotary_heads_backward(ctypes.byref(c.d), dev.stream), dev.lib)
    for (part, x, g, w, dw), dx in zip(c.parts, dxs):
        wh = w.double().cpu().numpy()
        want, dweight = ops.heads_gradient(x.host, g.host, c.at, c.radians, False, c.mag, True, wh, eps=0.0)
        size = pair_size(g.host, len(c.radians), False, c.mag)
        rms = np.sqrt((x.host ** 2).mean(-1, keepdims=True))
        y, t = np.abs(x.host / rms), size * np.abs(wh)
        err = (t + 3 * y * (t * y).mean(-1, keepdims=True)) / rms * 2 * NORM + np.abs(want) * 1.01 * ROUND[type] + TINY[type]
        assert (np.abs(dx.get() - want) <= err).all()
        n, total = want[..., 0].size, (size * y).reshape(-1, D).sum(0)
        assert (np.abs(dw.double().cpu().numpy() - dweight) <= total * (2 * NORM + (n / 32 + 64) * U)).all()


# ------------------------------------------------- sequences without any keys

@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("page,D", [(5, 64), (16, 128)])
@pytest.mark.parametrize("empty", [(1, 0), (3, 0), (20, 1)])
def test_runs_of_sequences_without_keys(dev, type, page, D, empty):
    """Tiles without keys, eight in a row and more than four a CTA, behind one with a last block that is not whole."""
    batch = ([(2, 134), (1, 60)] + [empty] * 4) * 70
    c = Cache(dev, batch, 2, D, page, type)
    check(dev, c, attend(dev, c, 66, max_new=20))


# ------------------------------------------- captured, far apart, very many

def captured(dev, call):
    """`call(stream)` captured into a graph; replay() launches it and waits."""
    t = dev.torch
    side, graph = t.cuda.Stream(), ctypes.c_void_p()
    stream = ctypes.c_void_p(side.cuda_stream)
    t.cuda.synchronize()
    capi.check(dev.lib.tl_graph_capture_begin(stream), dev.lib)
    call(stream)
    capi.check(dev.lib.tl_graph_capture_end(stream, ctypes.byref(graph)), dev.lib)

    def replay():
        t.cuda.synchronize()
        capi.check(dev.lib.tl_graph_launch(graph, stream), dev.lib)
        t.cuda.synchronize()

    return replay, lambda: capi.check(dev.lib.tl_graph_destroy(graph), dev.lib)


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
def test_a_captured_chunk_follows_values_that_are_not_finite(dev, type):
    """A replayed call sees a later token's infinite value come and go, and lengths that shrink."""
    c = Cache(dev, [(70, 600), (40, 300)], 2, 64, 16, type)
    s = attend(dev, c, 6, prepare_only=True)
    replay, close = captured(dev, lambda st: capi.check(dev.lib.tl_paged_attention(ctypes.byref(s["d"]), st), dev.lib))
    page, slot = c.places(0, 590, 591)
    good, kept = c.v[page, slot].clone(), c.vals[0][590].copy()
    full = c.batch, c.keys, c.vals
    for bad, keys in ((None, (600, 300)), (float("inf"), (600, 300)), (None, (600, 300)), (float("nan"), (595, 40)), (None, (70, 41))):
        c.v[page, slot] = good if bad is None else bad
        full[2][0][590] = kept if bad is None else bad
        c.c_lengths.copy_(dev.torch.tensor(keys).to(dev.torch.int32).view(c.c_lengths.dtype))
        c.batch = [(70, keys[0]), (40, keys[1])]
        c.keys, c.vals = ([x[i][:n] for i, n in enumerate(keys)] for x in full[1:])
        replay()
        check(dev, c, s)
    close()


@pytest.mark.parametrize("type", ["f32", "bf16"])
def test_a_captured_append_follows_the_lengths(dev, type):
    c = Cache(dev, [(3, 3), (1, 2), (20, 20)], 2, 64, 16, type)
    k, v = c.k.clone(), c.v.clone()
    s = append(dev, c, 4, 64, type, norm=True)  # once outside, for the oracle's numbers
    replay, close = captured(dev, lambda st: capi.check(dev.lib.tl_cache_append(ctypes.byref(s["d"]), st), dev.lib))
    for lengths in ((3, 2, 20), (9, 7, 31), (16, 1, 32)):
        c.k.copy_(k)
        c.v.copy_(v)
        s["q_out"].fill_(GUARD)
        c.c_lengths.copy_(dev.torch.tensor(lengths).to(dev.torch.int32).view(c.c_lengths.dtype))
        c.batch = [(n, length) for (n, _), length in zip(c.batch, lengths)]
        replay()
        check_append(dev, c, s, k, v)
        assert dev.status() == 0
    close()


@pytest.mark.parametrize("type,new", [("bf16", 2), ("bf16", 30), ("f32", 2)])
def test_queries_and_outputs_behind_32_bits(dev, type, new):
    """Rows of queries and outputs farther apart than 2^32 elements in all."""
    t = dev.torch
    c = Cache(dev, [(new, 90)], 1, 64, 16, type)
    stride = ((1 << 32) // new + 64) // 64 * 64
    rows = [t.empty(stride * (new - 1) + 128, dtype=torch_type(dev, type), device=dev.dev).as_strided((new, 2, 64), (stride, 64, 1))
            for _ in range(2)]
    rows[0].copy_(t.from_numpy(c.rng.standard_normal((new, 2, 64))))
    rows[1].fill_(GUARD)
    s = attend(dev, c, 2, q=rows[0], prepare_only=True)
    s["out"] = rows[1]
    s["d"].out = capi.TlHeadView(rows[1].data_ptr(), 0, 64, stride)
    capi.check(dev.lib.tl_paged_attention(ctypes.byref(s["d"]), dev.stream), dev.lib)
    check(dev, c, s)


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("max_new", [0, 2])
def test_a_hundred_thousand_sequences(dev, type, max_new):
    """One page each, most with one new token: the whole batch against the same sums by torch in 64 bits."""
    t, n, D = dev.torch, 100003, 8
    c = Cache(dev, [(1, 1)], 1, D, 4, type)
    rng = np.random.default_rng(8)
    new = rng.choice([0, 1, 1, 1, 2], n)
    keys = new + rng.integers(0, 3, n)
    c.k, c.v = (t.from_numpy(rng.standard_normal((n, 4, 1, D))).to(dev.dev).to(torch_type(dev, type)) for _ in range(2))
    c.pages, c.table, starts = n, rng.permutation(n)[:, None].astype(np.uint32), np.concatenate(([0], np.cumsum(new)))
    c.tokens, c.batch = int(starts[-1]), [(1, 1)] * n
    c.c_table, c.c_starts, c.c_lengths = (dev.t(x, np.uint32) for x in (c.table, starts, keys))
    s = attend(dev, c, 9, max_new=max_new)
    of = np.repeat(np.arange(n), new)
    position = keys[of] - new[of] + np.arange(c.tokens) - starts[of]
    at = t.from_numpy(c.table[of, 0].astype(np.int64)).to(dev.dev)
    k, v, q = c.k[at, :, 0].double(), c.v[at, :, 0].double(), s["q"].double()
    x = t.einsum("thd,tsd->ths", q, k) * s["d"].scale
    x = x.masked_fill((t.arange(4)[None] > t.from_numpy(position)[:, None]).to(dev.dev)[:, None], -math.inf)
    p, size = x.softmax(-1), t.einsum("ths,tsd->thd", x.softmax(-1), v.abs())
    products = s["d"].scale * t.einsum("thd,tsd->ths", q.abs(), k.abs()).amax(-1)
    rel = 2 * products * (D * U + 3 * U) + 2.0 ** -20 + 64 * U + (0 if type == "f32" else ROUND[type])
    want = t.einsum("ths,tsd->thd", p, v)
    assert ((s["out"].double() - want).abs() <= size * rel[..., None] + want.abs() * ROUND[type] + TINY[type]).all()
    assert ((s["lse"].double() - x.logsumexp(-1)).abs() <= rel + 2 * U * x.abs().nan_to_num(posinf=0).amax(-1)).all()
    assert dev.status() == 0


@pytest.mark.parametrize("width", [64, 65, 300])
def test_chunks_with_room_for_very_long_sequences(dev, width):
    """Pages of 2^20 slots and tables for 2^26 keys and more."""
    c = Cache(dev, [(70, 300), (2, 40)], 1, 8, 1 << 20, "bf16", spare=0)
    c.table = np.concatenate([c.table[:, :1], np.full((2, width - 1), 0xffffffff, np.uint32)], 1)
    c.c_table = dev.t(c.table, np.uint32)
    check(dev, c, attend(dev, c, 4))


# ------------------------------------------------------ sequences that are cut

@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("new,keys,cut", [(1, 100, 90), (3, 100, 98), (3, 100, 90), (40, 100, 80), (200, 300, 150), (3, 5000, 4999)])
@pytest.mark.parametrize("window", [0, 20])
def test_cut_sequences_keep_their_positions(dev, type, new, keys, cut, window):
    """The keys behind max_length are not there; the tokens' positions are as they were."""
    c = Cache(dev, [(new, keys), (1, 30)], 2, 64, 16, type)
    s = attend(dev, c, 4, 1, window, max_length=cut)
    dev.torch.cuda.synchronize()
    assert dev.status() == capi.TL_FLAG_INDEX_RANGE
    q, out, lse = (s[n].double().cpu().numpy() for n in ("q", "out", "lse"))
    for i in range(new):
        p = keys - new + i
        b = min(p + 1, cut)
        a = min(max(0, p + 1 - window), b) if window else 0
        want, wlse, size = (x[0] for x in ops.attention(q[i:i + 1], c.keys[0][a:b], c.vals[0][a:b], s["d"].scale, causal=False))
        most = np.abs(c.keys[0]).max(0).repeat(2, 0)  # a key head for two query heads
        ds = s["d"].scale * (np.abs(q[i]) * most).sum(-1) * (64 * U + 3 * U)
        longs = 2.0 ** -20 + (keys / 64 + 64) * U
        err = size * (2 * ds + longs + (0 if type == "f32" else ROUND[type]))[:, None] + np.abs(want) * ROUND[type] + TINY[type]
        assert (np.abs(out[i] - want) <= err).all(), i
        none = np.isneginf(wlse)
        assert (np.isneginf(lse[i]) == none).all() and (out[i][none] == 0).all()
        assert (np.abs(lse[i][~none] - wlse[~none]) <= (ds + longs + 2 * U * np.abs(wlse))[~none]).all(), i


# --------------------------------------------------------- fp32 products

@pytest.mark.parametrize("D", [64, 128, 40])
@pytest.mark.parametrize("batch", [[(1, 1), (3, 3), (1, 16)], [(40, 200), (1, 900)]])
@pytest.mark.parametrize("sharp", [1.0, 20.0])
def test_fp32_attention_in_fp32(dev, D, batch, sharp):
    """fp32 caches by fp32 products alone: a score is four lanes' four sums of D / 16 products, added up in four
    steps, so within S = (D / 16 + 4) u scale sum |q k| of itself, with each row's own sum; log2(e), the maximum and
    their difference round it by 4 u |s|, an exponential by 2^-22 of itself, numerators and sum alike.  The sums over
    keys and the warps' and parts' joins are chains of at most L / 32 + 24 roundings."""
    c = Cache(dev, batch, 2, D, 16, "f32")
    s = attend(dev, c, 4, sharp=sharp)
    out, lse, q = (s[n].double().cpu().numpy() for n in ("out", "lse", "q"))
    steps = (64 if D <= 64 else 128) / 16 + 4
    for i, (new, keys) in enumerate(batch):
        at = slice(int(c.starts[i]), int(c.starts[i]) + new)
        want, wlse, size = ops.attention(q[at], c.keys[i], c.vals[i], s["d"].scale)
        for r in range(new):
            k = c.keys[i][:keys - new + r + 1].repeat(2, 1)
            products = s["d"].scale * np.einsum("hd,lhd->hl", np.abs(q[at][r]), np.abs(k)).max(-1)
            ds, longs = (steps + 4) * U * products, 2.0 ** -22 + (keys / 32 + 24) * U
            err = size[r] * 2 * (ds + longs)[:, None] + 2 * U * np.abs(want[r])
            assert (np.abs(out[at][r] - want[r]) <= err).all(), (i, r)
            assert (np.abs(lse[at][r] - wlse[r]) <= ds + longs + 2 * U * np.abs(wlse[r])).all(), (i, r)


# --------------------------------------------------------------------- writer

@pytest.mark.parametrize("type,cache_type", [("f16", "bf16"), ("bf16", "f16")])
@pytest.mark.parametrize("D,rotary,interleaved", [(64, 64, False), (128, 64, True), (80, 0, False), (13, 6, False), (256, 256, True)])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("queries", [True, False])
def test_append_to_the_other_16_bit_type(dev, type, cache_type, D, rotary, interleaved, norm, queries):
    batch = [(3, 3), (1, 40), (0, 7), (20, 33), (0, 0), (1, 1)]
    for page, order, pad in ((16, "pshd", 0), (5, "phsd", 8), (1, "interleaved", 3)):
        c = Cache(dev, batch, 2, D, page, cache_type, order, extra=3, gaps=True)
        k, v = c.k.clone(), c.v.clone()
        s = append(dev, c, 5, rotary, type, None, interleaved, norm, pad, queries=queries)
        check_append(dev, c, s, k, v, queries=queries)
        assert dev.status() == 0


@pytest.mark.parametrize("what", ["backwards", "behind", "all_behind", "length", "empty_length"])
def test_append_raises_the_flag_for_every_bad_sequence(dev, what):
    """Also for those that no row of the call leads to; the others are written."""
    c = Cache(dev, [(3, 50)] if what == "backwards" else [(2, 40), (0, 30), (3, 50)], 2, 64, 16, "bf16", extra=5)
    if what == "backwards":       # rows 5 .. 3
        skip, starts = (0,), [5, 3]
    elif what == "behind":        # the last one's rows end behind the tensors
        skip, starts = (2,), [0, 2, 2, c.tokens + 1]
    elif what == "all_behind":    # they lie behind the tensors altogether
        skip, starts = (2,), [0, 2, c.tokens, c.tokens + 3]
        c.batch[1] = (c.tokens - 2, 30)
    else:                         # more keys than a row of the table holds, with and without new tokens
        skip, starts = (2 if what == "length" else 1,), [0, 2, 2, 5]
        c.c_lengths[skip[0]] = c.table.shape[1] * c.page + 1
    c.c_starts = dev.t(starts, np.uint32)
    k, v = c.k.clone(), c.v.clone()
    s = append(dev, c, 2, 64, "bf16")
    dev.torch.cuda.synchronize()
    assert dev.status() == capi.TL_FLAG_INDEX_RANGE
    check_append(dev, c, s, k, v, skip=skip)
