"""Rotation and norm of heads (tl_rotary_heads, its gradient) against the
float64 oracle (oracle/head_ops.py) on the inputs as the kernels hold them.

Tolerances, from the arithmetic (u = 2^-24, fp32's rounding).  Angles are
exact to 2^-62 of a turn; the rest of a quarter turn is rounded twice, the
series adds 2.5e-8 < u / 2 and its sum u, the magnitude u: a sine or cosine is
within 5 u of itself (of 1), and a cos - b sin within 7 u (|a| + |b|)
magnitude.  The norm: a sum of D / lanes + log2(lanes) <= 36 + 5 rounded terms,
whose root halves the error, the root's and two products' roundings: 24 u.
NORM is both.  The gradient subtracts x^ mean(g x^): three such errors of
sizes that max |g w| bounds.  The result's rounding: half a unit of its type.
A weight's gradient sums n terms, each within 2 NORM of its size, in runs
of at most n / 32 + 64."""
import ctypes

import numpy as np
import pytest

from oracle import head_ops as ops
from templit_b200 import capi
from tests.helpers import Dev

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
ROUND = {"f32": U, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -133}
TYPES = {"f32": capi.TL_FLOAT32, "f16": capi.TL_FLOAT16, "bf16": capi.TL_BFLOAT16}
TURN, NORM = 8 * U, 32 * U
GUARD = 7.0


@pytest.fixture(scope="module")
def dev():
    return Dev()


def torch_type(dev, type):
    return {"f32": dev.torch.float32, "f16": dev.torch.float16, "bf16": dev.torch.bfloat16}[type]


class Heads:
    """[B, T, H, D] values in one of several memory orders, with GUARD around them."""

    def __init__(self, dev, values, type, order="bthd", pad=0, offset=0):
        self.dev, self.type, self.order, self.pad, self.offset = dev, type, order, pad, offset
        B, T, H, D = values.shape
        axes = {"bthd": (0, 1, 2), "bhtd": (0, 2, 1), "tbhd": (1, 0, 2)}[order]
        shape = [values.shape[i] for i in axes]
        self.buf = dev.torch.full((offset + int(np.prod(shape)) * (D + pad) + 16,), GUARD,
                                  dtype=torch_type(dev, type), device=dev.dev)
        flat = self.buf[offset:offset + int(np.prod(shape)) * (D + pad)].view(*shape, D + pad)[..., :D]
        self.view = flat.permute(*np.argsort(axes).tolist(), 3)
        self.view.copy_(dev.torch.from_numpy(np.ascontiguousarray(values)))
        self.host = self.view.double().cpu().numpy()

    def like(self, type=None):
        return Heads(self.dev, np.full(self.view.shape, GUARD), type or self.type, self.order, self.pad, self.offset)

    def c(self):
        s = self.view.stride()
        return capi.TlHeadView(self.view.data_ptr(), s[0], s[2], s[1])

    def get(self):
        """Values; nothing around them may have changed."""
        out = self.view.double().cpu().numpy()
        keep = self.view.clone()
        self.view.fill_(GUARD)
        assert (self.buf == GUARD).all()
        self.view.copy_(keep)
        return out


def table(dev, dim, **kw):
    """Frequencies as the library gives them, and the oracle's radians."""
    names = {"scaling": "scaling", "factor": "factor", "original": "original_length", "low": "low", "high": "high"}
    spec = capi.TlRotarySpec(dim=dim, base=kw.get("base", 10000.0), **{names[k]: v for k, v in kw.items() if k in names})
    out, mag = (ctypes.c_uint64 * (dim // 2))(), ctypes.c_float()
    capi.check(dev.lib.tl_rotary_frequencies(ctypes.byref(spec), out, ctypes.byref(mag)), dev.lib)
    radians, _ = ops.frequencies(dim, **kw)
    return dev.torch.frombuffer(bytearray(out), dtype=dev.torch.int64).to(dev.dev), mag.value, radians


class Case:
    def __init__(self, dev, B, T, hq, hk, D, rotary, type="f32", out_type=None, interleaved=False, norm=False,
                 weighted=True, positions=None, first=0, order="bthd", pad=0, offset=0, seed=0, scale=1.0, **freq):
        rng = np.random.default_rng(seed)
        self.dev, self.out_type, self.norm, self.interleaved = dev, out_type or type, norm, interleaved
        self.D, self.type, self.B, self.T = D, type, B, T
        if rotary:
            self.frequencies, self.mag, self.radians = table(dev, rotary, **freq)
        else:
            self.frequencies, self.mag, self.radians = None, 1.0, np.zeros(0)
        self.at = np.broadcast_to(first + np.arange(T), (B, T)) if positions is None else positions(rng, (B, T))
        self.positions = None if positions is None else dev.t(self.at, np.uint32)
        d = self.d = capi.TlRotaryDesc(B=B, T=T, D=D, rotary_dim=rotary, type=TYPES[type], out_type=TYPES[self.out_type],
                                       layout=int(interleaved), norm=int(norm), eps=1e-6, magnitude=self.mag,
                                       frequencies=self.frequencies.data_ptr() if rotary else None,
                                       positions=self.positions.data_ptr() if positions else None, first_position=first)
        self.parts = []
        for part, h in ((d.q, hq), (d.k, hk)):
            part.heads = h
            if not h:
                continue
            x = Heads(dev, rng.standard_normal((B, T, h, D)) * scale, type, order, pad, offset)
            g = Heads(dev, rng.standard_normal((B, T, h, D)), self.out_type, order, pad, offset)
            w = dev.t(1 + 0.3 * rng.standard_normal(D)) if norm and weighted else None
            dw = dev.t(np.full(D, GUARD)) if norm and weighted else None
            part.x, part.d_out = x.c(), g.c()
            part.weight, part.dweight = dev.p(w), dev.p(dw)
            self.parts.append((part, x, g, w, dw))

    def forward(self, in_place=False):
        outs = []
        for part, x, *_ in self.parts:
            outs.append(x if in_place else x.like(self.out_type))
            part.out = outs[-1].c()
        capi.check(self.dev.lib.tl_rotary_heads(ctypes.byref(self.d), self.dev.stream), self.dev.lib, "tl_rotary_heads")
        for (part, x, g, w, dw), out in zip(self.parts, outs):
            kw = dict(interleaved=self.interleaved, magnitude=self.mag)
            wh = None if w is None else w.double().cpu().numpy()
            want = ops.heads(x.host, self.at, self.radians, normed=self.norm, weight=wh, **kw)
            y = ops.norm(x.host, wh) if self.norm else x.host
            size = pair_size(y, len(self.radians), self.interleaved, self.mag)
            got = out.get()
            assert got.shape == want.shape
            err = size * (NORM if self.norm else TURN) + np.abs(want) * 1.01 * ROUND[self.out_type] + TINY[self.out_type]
            if not self.norm:  # what is not turned is copied, rounded at most
                err[..., 2 * len(self.radians):] = (np.abs(want) * ROUND[self.out_type] + TINY[self.out_type])[..., 2 * len(self.radians):]
            worst = (np.abs(got - want) / err).max()
            assert worst <= 1, worst
        return outs

    def backward(self, in_place=False):
        dxs = []
        for part, x, g, *_ in self.parts:
            dxs.append(g if in_place else x.like())
            part.dx = dxs[-1].c()
        lib = self.dev.lib
        ws = self.dev.ws(lib.tl_rotary_heads_workspace_size(ctypes.byref(self.d)))
        self.d.workspace, self.d.workspace_bytes = ws.data_ptr(), ws.numel()
        self.hold = (ws, dxs)  # a captured call writes there again
        capi.check(lib.tl_rotary_heads_backward(ctypes.byref(self.d), self.dev.stream), lib, "tl_rotary_heads_backward")
        for (part, x, g, w, dw), dx in zip(self.parts, dxs):
            wh = None if w is None else w.double().cpu().numpy()
            want, dweight = ops.heads_gradient(x.host, g.host, self.at, self.radians, self.interleaved, self.mag,
                                               self.norm, wh)
            size = pair_size(g.host, len(self.radians), self.interleaved, self.mag)
            if self.norm:
                rms = np.sqrt((x.host ** 2).mean(-1, keepdims=True) + 1e-6)
                y = np.abs(x.host / rms)
                t = size * (1 if wh is None else np.abs(wh))
                err = (t + 3 * y * (t * y).mean(-1, keepdims=True)) / rms * 2 * NORM
            else:
                err = size * TURN
            err = err + np.abs(want) * 1.01 * ROUND[self.type] + TINY[self.type]
            got = dx.get()
            worst = (np.abs(got - want) / err).max()
            assert worst <= 1, worst
            if dw is not None:
                n = want[..., 0].size
                total = (size * y).reshape(-1, self.D).sum(0)
                assert (np.abs(dw.double().cpu().numpy() - dweight) <= total * (2 * NORM + (n / 32 + 64) * U)).all()


def pair_size(x, half, interleaved, mag):
    """|a| + |b| at both elements of a pair, |x| behind."""
    x = np.abs(np.asarray(x, np.float64))
    out = x.copy()
    i = np.arange(half)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    out[..., a] = out[..., b] = (x[..., a] + x[..., b]) * abs(mag)
    return out


SHAPES = [(1, 1, 6, 6, 64, 64), (2, 5, 4, 1, 128, 128), (3, 7, 5, 2, 128, 64), (1, 33, 3, 3, 32, 32), (2, 9, 7, 1, 256, 256),
          (1, 4, 2, 2, 80, 40), (1, 3, 1, 9, 8, 8), (2, 3, 2, 1, 65, 64), (1, 5, 3, 2, 13, 6), (1, 2, 1, 1, 2, 2),
          (1, 2, 2, 3, 1, 0), (1, 6, 3, 1, 96, 0), (2, 3, 0, 4, 64, 32), (1, 3, 5, 0, 112, 112), (1, 2, 3, 2, 251, 250)]


@pytest.mark.parametrize("B,T,hq,hk,D,rotary", SHAPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("norm", [False, True])
def test_shapes(dev, B, T, hq, hk, D, rotary, interleaved, type, norm):
    c = Case(dev, B, T, hq, hk, D, rotary, type, interleaved=interleaved, norm=norm, first=11)
    c.forward()
    c.backward()


@pytest.mark.parametrize("type,out_type", [("f32", "bf16"), ("f32", "f16"), ("bf16", "f32"), ("f16", "f32")])
@pytest.mark.parametrize("D,rotary", [(64, 64), (128, 32), (40, 12)])
@pytest.mark.parametrize("norm", [False, True])
def test_two_types(dev, type, out_type, D, rotary, norm):
    c = Case(dev, 2, 5, 4, 2, D, rotary, type, out_type, norm=norm)
    c.forward()
    c.backward()


@pytest.mark.parametrize("order", ["bthd", "bhtd", "tbhd"])
@pytest.mark.parametrize("pad,offset", [(0, 0), (8, 8), (3, 0), (0, 1), (5, 7)])
@pytest.mark.parametrize("type", ["f32", "bf16"])
def test_orders_and_alignments(dev, order, pad, offset, type):
    c = Case(dev, 3, 5, 4, 2, 64, 64, type, norm=True, order=order, pad=pad, offset=offset)
    c.forward()
    c.backward()


@pytest.mark.parametrize("freq", [dict(), dict(scaling=ops.LINEAR, factor=4.0), dict(scaling=ops.NTK, factor=8.0),
                                  dict(scaling=ops.PARTS, factor=8.0, original=4096.0, low=1.0, high=32.0),
                                  dict(scaling=ops.SMOOTH, factor=8.0, original=8192.0, low=1.0, high=4.0),
                                  dict(base=1e6)])
@pytest.mark.parametrize("far", [1000, 1 << 20, (1 << 32) - 1])
def test_far_positions(dev, freq, far):
    """The oracle's own angles round at 2^-53 * 2^32 turns = 2^-21 of a turn for the farthest positions: it gets
    them from whole numbers instead."""
    c = Case(dev, 2, 16, 2, 1, 64, 64, "f32", positions=lambda rng, s: rng.integers(0, far, s, endpoint=True, dtype=np.uint64),
             **freq)
    turns = [int(x) & (2 ** 64 - 1) for x in c.frequencies.cpu().numpy()]
    angle = np.array([[[(int(p) * f % 2 ** 64) / 2.0 ** 64 * 2 * np.pi for f in turns] for p in row] for row in c.at])
    outs = []
    for part, x, *_ in c.parts:
        outs.append(x.like())
        part.out = outs[-1].c()
    capi.check(dev.lib.tl_rotary_heads(ctypes.byref(c.d), dev.stream), dev.lib)
    for (part, x, *_), out in zip(c.parts, outs):
        a, b = x.host[..., :32], x.host[..., 32:]
        cos, sin = c.mag * np.cos(angle)[:, :, None], c.mag * np.sin(angle)[:, :, None]
        want = np.concatenate((a * cos - b * sin, a * sin + b * cos), -1)
        size = pair_size(x.host, 32, False, c.mag)
        assert (np.abs(out.get() - want) <= size * TURN + np.abs(want) * U).all()


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("D,rotary", [(64, 64), (13, 6)])
def test_in_place(dev, type, D, rotary):
    c = Case(dev, 2, 7, 4, 2, D, rotary, type, norm=True, weighted=False)
    c.backward(in_place=True)
    c.forward(in_place=True)


def test_without_weights(dev):
    c = Case(dev, 2, 5, 3, 2, 128, 128, "bf16", norm=True, weighted=False)
    c.forward()
    c.backward()


def test_rows_of_zeros_and_large_numbers(dev):
    for scale in (0.0, 1e-18, 1e15):
        c = Case(dev, 1, 5, 2, 1, 64, 64, "f32", norm=True, scale=scale)
        c.forward()


def test_nan_stays_in_its_head(dev):
    c = Case(dev, 1, 4, 3, 1, 64, 32, "f32", norm=True)
    x = c.parts[0][1]
    x.view[0, 2, 1, 40] = float("nan")
    out = x.like()
    c.d.q.out = out.c()
    c.d.k.heads = 0
    capi.check(dev.lib.tl_rotary_heads(ctypes.byref(c.d), dev.stream), dev.lib)
    bad = np.isnan(out.get())
    assert bad[0, 2, 1].all() and bad.sum() == 64


@pytest.mark.parametrize("B,T,hq,hk,D", [(4, 700, 12, 3, 128), (1, 5000, 1, 1, 64), (1, 4000, 13, 5, 128), (2, 3001, 9, 7, 96),
                                         (1, 3500, 21, 10, 40)])
@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
def test_many_tokens(dev, B, T, hq, hk, D, type):
    """More work than one round of the grid, heads that do not fill a warp's last batch: weight gradients over all of it."""
    c = Case(dev, B, T, hq, hk, D, D, type, norm=True)
    c.forward()
    c.backward()


def test_broadcast_input(dev):
    """One row of keys for every head and batch (strides of 0)."""
    c = Case(dev, 3, 4, 5, 1, 64, 64, "f32")
    part, x, *_ = c.parts[0]
    part.x = capi.TlHeadView(x.view.data_ptr(), 0, 0, x.view.stride(1))
    x.host = np.broadcast_to(x.host[:1, :, :1], x.host.shape)
    c.forward()


def test_no_tokens_clear_the_weight_gradients(dev):
    c = Case(dev, 1, 2, 2, 2, 64, 64, norm=True)
    ws = dev.ws(dev.lib.tl_rotary_heads_workspace_size(ctypes.byref(c.d)))
    c.d.workspace, c.d.workspace_bytes, c.d.T = ws.data_ptr(), ws.numel(), 0
    capi.check(dev.lib.tl_rotary_heads_backward(ctypes.byref(c.d), dev.stream), dev.lib)
    for part, x, g, w, dw in c.parts:
        assert (dw == 0).all()


def test_same_result_every_time_and_in_a_graph(dev):
    torch = dev.torch
    c = Case(dev, 3, 400, 8, 2, 128, 128, "bf16", norm=True)
    c.backward()
    first = [(p[4].clone()) for p in c.parts]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = ctypes.c_void_p()
    s = ctypes.c_void_p(side.cuda_stream)
    capi.check(dev.lib.tl_graph_capture_begin(s), dev.lib)
    capi.check(dev.lib.tl_rotary_heads_backward(ctypes.byref(c.d), s), dev.lib)
    capi.check(dev.lib.tl_graph_capture_end(s, ctypes.byref(graph)), dev.lib)
    for _ in range(3):
        for p in c.parts:
            p[4].fill_(GUARD)
        torch.cuda.synchronize()
        capi.check(dev.lib.tl_graph_launch(graph, s), dev.lib)
        side.synchronize()
        assert all((a == p[4]).all() for a, p in zip(first, c.parts))
    capi.check(dev.lib.tl_graph_destroy(graph), dev.lib)
