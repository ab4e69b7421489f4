"""Measured workloads of the rotation, head norm, cache and paged attention operators.

Four entry points of include/templit_cuda.h:

  rotate       tl_rotary_heads: queries and keys turned by their positions; with `norm`, each head
               normed (RMS, a weight per element) in the same pass
  rotate_grad  tl_rotary_heads_backward: its gradient (with `norm`: the weights' too)
  append       tl_cache_append: new keys (turned, normed) and values into a paged cache, queries alike
  attend       tl_paged_attention: new tokens of every sequence over its keys and values in the cache

`own` chooses between the plain form (elementary torch operations in 32 bits, angles in 64) and the
kernels.  6 heads of 64, T = 192 and batches of 64 are the framework's own model; grouped heads, long
caches and long chunks are generic.
"""
import ctypes
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
KINDS = ("rotate", "rotate_grad", "append", "attend", "attend")
EPS = 1e-6
ELEMENTS = 16384 * 40 * 128      # heads' elements of the largest listed rotation
FLOPS = 4 * 128 * 32 * 8192 * 4096  # of the largest listed attention
KEYS = 200003 * 8 * 128          # key elements of the largest listed cache


def _heads(name, kind, tokens, q_heads, kv_heads, dim, type, **more):
    c = {"name": name, "kind": kind, "batch": 1, "tokens": tokens, "q_heads": q_heads, "kv_heads": kv_heads,
         "dim": dim, "rotary": dim, "type": type, "layout": "half", "scaling": "plain", "norm": False, "far": 0}
    c.update(more)
    return c


def _cache(name, kind, sequences, new, keys, q_heads, kv_heads, dim, type, page, **more):
    """`new` tokens and `keys` keys (those included) in the longest sequence; ragged: shorter ones too."""
    c = {"name": name, "kind": kind, "sequences": sequences, "new": new, "keys": keys, "q_heads": q_heads,
         "kv_heads": kv_heads, "dim": dim, "type": type, "page": page, "ragged": True, "window": 0}
    if kind == "append":
        c.update({"rotary": dim, "layout": "half", "scaling": "plain", "norm": False, "from": type})
    c.update(more)
    return c


def listed():
    return [
        # queries and keys of the framework's training batch: 64 sequences of 192 tokens
        _heads("rotate_train_batch", "rotate", 192, 6, 6, 64, "f32", batch=64),
        # the backward pass of half-turned heads, adjacent pairs, a context stretched by parts
        _heads("rotate_grad_partial", "rotate_grad", 2048, 32, 8, 128, "f16", batch=8, rotary=64,
               layout="interleaved", scaling="parts"),
        # one generated token of 64 sequences: norm and rotation
        _heads("norm_step_64", "rotate", 64, 32, 8, 128, "bf16", norm=True, far=100000),
        # norm and rotation of a long batch
        _heads("norm_batch", "rotate", 16384, 32, 8, 128, "bf16", norm=True),
        # its gradient
        _heads("norm_grad_batch", "rotate_grad", 16384, 32, 8, 128, "bf16", norm=True),
        # one generated token of 64 sequences into the cache
        _cache("append_step_64", "append", 64, 1, 4099, 32, 8, 128, "bf16", 16, norm=True),
        # chunks of prompts, from the products' 32 bits into a 16-bit cache
        _cache("append_chunks", "append", 16, 1000, 2003, 32, 8, 128, "bf16", 16, **{"from": "f32"}),
        # one generated token of the framework's own model at the end of its window
        _cache("attend_one_token", "attend", 1, 1, 192, 6, 6, 64, "f32", 16, ragged=False),
        # one decoding step of 64 sequences of very different lengths
        _cache("attend_step_64", "attend", 64, 1, 8191, 32, 8, 128, "bf16", 16),
        # one token of one long conversation
        _cache("attend_step_long", "attend", 1, 1, 200003, 32, 8, 128, "bf16", 64, ragged=False),
        # prompts in chunks beside decoding sequences, odd group of heads
        _cache("attend_chunks", "attend", 24, 509, 4093, 24, 8, 64, "f16", 16),
        # a long prompt at once
        _cache("attend_prompt", "attend", 1, 8192, 8192, 32, 8, 128, "bf16", 64, ragged=False),
    ]


def draw(rng):
    spread = lambda a, b: int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))  # noqa: E731
    kind = rng.choice(KINDS)
    kv_heads = rng.choice((1, 2, 3, 4, 6, 8))
    q_heads = kv_heads * rng.choice((1, 1, 2, 3, 4, 7, 8))
    dim = rng.choice((64, 128, 64, 128, 32, 40, 80, 96, 112))
    type = rng.choice(("f32", "f16", "bf16", "bf16"))
    turn = {"rotary": rng.choice((dim, dim, dim // 4 * 2)), "layout": rng.choice(("half", "interleaved")),
            "scaling": rng.choice(("plain", "linear", "ntk", "parts", "smooth")), "norm": rng.random() < 0.5}
    if kind in ("rotate", "rotate_grad"):
        batch = rng.choice((1, 1, spread(1, 64)))
        most = ELEMENTS // ((q_heads + kv_heads) * dim * batch * (2 if type == "f32" else 1))
        return _heads(None, kind, max(1, min(spread(1, 16384), most)), q_heads, kv_heads, dim, type, batch=batch,
                      far=rng.choice((0, spread(1, 4000000))), **turn) | {"name": ""}
    sequences, new = spread(1, 128), rng.choice((1, 1, spread(1, 64), spread(1, 4096)))
    size = 2 if type == "f32" else 1
    new = max(1, min(new, 16384 * 8 // (sequences * (q_heads + 2 * kv_heads) * size)))
    keys = min(new + spread(1, 130000), max(new, KEYS // (kv_heads * dim * sequences * size)))
    if kind == "append":
        keys = min(keys, new + 4096)
        return _cache("", kind, sequences, new, keys, q_heads, kv_heads, dim, rng.choice(("f16", "bf16", type)),
                      rng.choice((16, 16, 64, 1, rng.randint(2, 200))), **turn, **{"from": type})
    # products of 32-bit numbers cost about sixteen times those of 16-bit ones
    cost = 4 * 128 * q_heads * sequences * (16 if type == "f32" else 1)
    if cost * new * keys > FLOPS:
        keys = max(new, FLOPS // (cost * new))
        new = max(1, min(new, FLOPS // (cost * keys)))
    return _cache("", kind, sequences, new, keys, q_heads, kv_heads, dim, type,
                  rng.choice((16, 16, 64, 1, rng.randint(2, 200))), ragged=rng.random() < 0.8,
                  window=rng.choice((0, 0, 0, spread(1, 4096))))


def _lengths(case):
    """(new tokens, keys) of every sequence, the same for every seed."""
    rng = random.Random(f"{case['sequences']} {case['new']} {case['keys']} {case['dim']}")
    out = []
    for s in range(case["sequences"]):
        if not case["ragged"] or s == 0:
            out.append((case["new"], case["keys"]))
            continue
        # decoding sequences among the prompts; lengths over their logarithm
        new = 1 if rng.random() < 0.5 else int(round(math.exp(rng.uniform(0, math.log(case["new"])))))
        out.append((new, max(new, int(round(math.exp(rng.uniform(math.log(16), math.log(case["keys"] + 16))))) - 16)))
    return out


def _seen(case, new, keys):
    """(query, key) pairs and keys that a sequence's new tokens see."""
    w, first = case["window"] or keys, keys - new
    pairs = sum(min(p + 1, w) for p in range(first, keys))
    return pairs, min(keys, new + w - 1)


def work(case):
    b, kind = BYTES[case["type"]], case["kind"]
    if kind in ("rotate", "rotate_grad"):
        n = case["batch"] * case["tokens"]
        e = n * (case["q_heads"] + case["kv_heads"]) * case["dim"]
        arrays = 3 if kind == "rotate_grad" and case["norm"] else 2
        return {"bytes": e * b * arrays + 4 * n + 4 * case["rotary"] + (8 * case["dim"] if case["norm"] else 0),
                "flops": e * (3 + (4 if case["norm"] else 0) * (2 if kind == "rotate_grad" else 1))}
    h, g, d = case["kv_heads"], case["q_heads"], case["dim"]
    if kind == "append":
        n = sum(new for new, _ in _lengths(case))
        return {"bytes": n * (g + 2 * h) * d * (BYTES[case["from"]] + b), "flops": n * (g + h) * d * (7 if case["norm"] else 3)}
    pairs = keys = n = 0
    for new, length in _lengths(case):
        p, k = _seen(case, new, length)
        pairs, keys, n = pairs + p, keys + k, n + new
    return {"bytes": (2 * keys * h + 2 * n * g) * d * b, "flops": pairs * g * (4 * d + 4)}


# ------------------------------------------------------------------ inputs

BASE, FACTOR, ORIGINAL = 10000.0, 8.0, 4096.0


def _frequencies(case):
    """Radians a position of every pair, in 64 bits, and the magnitude."""
    r, kind = case["rotary"], case["scaling"]
    i = torch.arange(r // 2, dtype=torch.float64)
    if kind == "ntk":
        return (BASE * FACTOR ** (r / (r - 2.0))) ** (-2 * i / r), 1.0
    f = BASE ** (-2 * i / r)
    if kind == "linear":
        return f / FACTOR, 1.0
    if kind == "parts":  # pairs that turn more than 32 times over the original length stay, fewer than once stretch
        pair = lambda turns: r * math.log(ORIGINAL / (turns * 2 * math.pi)) / (2 * math.log(BASE))  # noqa: E731
        lo, hi = max(math.floor(pair(32.0)), 0), min(math.ceil(pair(1.0)), r - 1)
        ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        return f * (1 - ramp) + f / FACTOR * ramp, 0.1 * math.log(FACTOR) + 1.0
    if kind == "smooth":  # the same by the number of turns, between 1 and 4
        part = ((ORIGINAL * f / (2 * math.pi) - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return f / FACTOR * (1 - part) + f * part, 1.0
    return f, 1.0


def _weights(case, gen, dev):
    return 1.0 + 0.2 * torch.randn(case["dim"], generator=gen, device=dev)


def _normal(gen, dev, type, *shape):
    return torch.randn(shape, generator=gen, device=dev).to(TYPES[type])


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    s = {"case": case}
    if case["kind"] in ("rotate", "rotate_grad", "append"):
        f, s["magnitude"] = _frequencies(case)
        s["radians"] = f.to(dev)
        if case["norm"]:
            s["q_weight"], s["k_weight"] = _weights(case, gen, dev), _weights(case, gen, dev)
    (_prepare_heads if case["kind"] in ("rotate", "rotate_grad") else _prepare_cache)(case, s, gen, dev)
    if own:
        s["call"], s["plan"] = _plan(s)
    return s


def _prepare_heads(case, s, gen, dev):
    b, t, d = case["batch"], case["tokens"], case["dim"]
    # one product gives queries and keys side by side in a row
    both = case["q_heads"] + case["kv_heads"]
    at = (lambda x: (x[:, :, :case["q_heads"]], x[:, :, case["q_heads"]:]))
    s["q"], s["k"] = at(_normal(gen, dev, case["type"], b, t, both, d).mul_(1.5))
    s["positions"] = None
    if case["far"]:
        s["positions"] = torch.randint(0, case["far"], (b, t), generator=gen, device=dev, dtype=torch.int32)
    empty = lambda: torch.empty(b, t, both, d, dtype=TYPES[case["type"]], device=dev)  # noqa: E731
    if case["kind"] == "rotate":
        s["q_out"], s["k_out"] = at(empty())
    else:
        s["dq_out"], s["dk_out"] = at(_normal(gen, dev, case["type"], b, t, both, d))
        s["dq"], s["dk"] = at(empty())
        if case["norm"]:
            s["dq_weight"], s["dk_weight"] = torch.empty(d, device=dev), torch.empty(d, device=dev)


def _prepare_cache(case, s, gen, dev):
    h, g, d, page = case["kv_heads"], case["q_heads"], case["dim"], case["page"]
    s["lengths"] = _lengths(case)
    need = [-(-keys // page) for _, keys in s["lengths"]]
    pages = sum(need) + 7
    order = torch.randperm(pages, generator=gen, device=dev, dtype=torch.int32)
    s["table"] = torch.zeros(case["sequences"], max(need) + 1, dtype=torch.int32, device=dev)
    used, starts = 0, [0]
    for i, n in enumerate(need):
        s["table"][i, :n] = order[used:used + n]
        used += n
        starts.append(starts[-1] + s["lengths"][i][0])
    s["starts_host"], n = starts, starts[-1]
    s["starts"] = torch.tensor(starts, dtype=torch.int32, device=dev)
    s["keys"] = torch.tensor([k for _, k in s["lengths"]], dtype=torch.int32, device=dev)
    s["k_cache"], s["v_cache"] = (_normal(gen, dev, case["type"], pages, page, h, d) for _ in range(2))
    if case["kind"] == "append":
        row = _normal(gen, dev, case["from"], n, g + 2 * h, d)
        s["q"], s["k"], s["v"] = row[:, :g], row[:, g:g + h], row[:, g + h:]
        s["q_out"] = torch.empty(n, g, d, dtype=TYPES[case["type"]], device=dev)
    else:
        # queries sharp enough that a few keys matter
        s["q"] = _normal(gen, dev, case["type"], n, g, d).mul_(2.0)
        s["out"] = torch.empty(n, g, d, dtype=TYPES[case["type"]], device=dev)
        s["lse"] = torch.empty(n, g, device=dev)


# --------------------------------------------------------------- plain form

def _cos_sin(s, positions):
    """[..., 1, rotary / 2] in 32 bits from angles in 64."""
    angle = positions.double()[..., None, None] * s["radians"]
    return (angle.cos() * s["magnitude"]).float(), (angle.sin() * s["magnitude"]).float()


def _turn(case, x, cos, sin):
    r = case["rotary"]
    out = x.clone()
    if case["layout"] == "half":
        a, b = slice(0, r // 2), slice(r // 2, r)
    else:
        a, b = slice(0, r, 2), slice(1, r, 2)
    out[..., a] = x[..., a] * cos - x[..., b] * sin
    out[..., b] = x[..., a] * sin + x[..., b] * cos
    return out


def _normed(x):
    return x * (1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS))


def _heads_positions(s):
    case = s["case"]
    if s["positions"] is not None:
        return s["positions"]
    return torch.arange(case["tokens"], device=s["q"].device).expand(case["batch"], -1)


def _rotate_plain(s):
    case, out = s["case"], {}
    cos, sin = _cos_sin(s, _heads_positions(s))
    for name in ("q", "k"):
        x = s[name].float()
        if case["norm"]:
            x = _normed(x) * s[name + "_weight"]
        out[name + "_out"] = _turn(case, x, cos, sin).to(s[name].dtype)
    return out


def _rotate_grad_plain(s):
    case, out = s["case"], {}
    cos, sin = _cos_sin(s, _heads_positions(s))
    for name in ("q", "k"):
        g = _turn(case, s[f"d{name}_out"].float(), cos, -sin)
        if case["norm"]:
            x = s[name].float()
            scale = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
            x = x * scale
            # a long sum: in 64 bits
            out[f"d{name}_weight"] = (g * x).sum((0, 1, 2), dtype=torch.float64).float()
            g = g * s[name + "_weight"]
            g = (g - x * (g * x).mean(-1, keepdim=True)) * scale
        out["d" + name] = g.to(s[name].dtype)
    return out


def _new_positions(s):
    dev = s["q"].device
    return torch.cat([torch.arange(keys - new, keys, device=dev) for new, keys in s["lengths"]])


def _append_plain(s):
    case = s["case"]
    positions = _new_positions(s)
    cos, sin = _cos_sin(s, positions)
    q, k = s["q"].float(), s["k"].float()
    if case["norm"]:
        q, k = _normed(q) * s["q_weight"], _normed(k) * s["k_weight"]
    counts = torch.tensor([new for new, _ in s["lengths"]], device=q.device)
    row = torch.repeat_interleave(torch.arange(len(s["lengths"]), device=q.device), counts, output_size=q.shape[0])
    page = s["table"][row, positions // case["page"]].long()
    slot = positions % case["page"]
    s["k_cache"][page, slot] = _turn(case, k, cos, sin).to(s["k_cache"].dtype)
    s["v_cache"][page, slot] = s["v"].to(s["v_cache"].dtype)
    return {"q_out": _turn(case, q, cos, sin).to(s["q_out"].dtype), "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _attend_plain(s):
    case = s["case"]
    h, g, d = case["kv_heads"], case["q_heads"] // case["kv_heads"], case["dim"]
    out, lse = torch.empty_like(s["out"]), torch.empty_like(s["lse"])
    for i, (new, keys) in enumerate(s["lengths"]):
        pages = s["table"][i, :-(-keys // case["page"])].long()
        k, v = (s[c][pages].reshape(-1, h, d)[:keys].float() for c in ("k_cache", "v_cache"))
        at = slice(s["starts_host"][i], s["starts_host"][i] + new)
        q = s["q"][at].float().view(new, h, g, d)
        own_at = torch.arange(keys - new, keys, device=q.device)
        key_at = torch.arange(keys, device=q.device)
        hidden = key_at[None, :] > own_at[:, None]
        if case["window"]:
            hidden |= key_at[None, :] <= own_at[:, None] - case["window"]
        step = max(1, (1 << 28) // (new * g * keys))  # heads at once
        for a in range(0, h, step):
            e = slice(a, a + step)
            x = torch.einsum("nhgd,khd->hngk", q[:, e], k[:, e]) * (1.0 / math.sqrt(d))
            x.masked_fill_(hidden[None, :, None, :], -math.inf)
            m = x.max(-1, keepdim=True).values
            p = (x - m).exp_()
            total = p.sum(-1, keepdim=True)
            o = torch.einsum("hngk,khd->nhgd", p, v[:, e]) / total.permute(1, 0, 2, 3)
            out[at].view(new, h, g, d)[:, e] = o.to(out.dtype)
            lse[at].view(new, h, g)[:, e] = (m + total.log())[..., 0].permute(1, 0, 2)
    return {"out": out, "lse": lse}


# ------------------------------------------------------------------ kernels

def _plan(s):
    """The call and its descriptor: the pointers and sizes that a program fills in once."""
    from templit_b200 import capi
    lib, case = capi.cuda_lib(), s["case"]
    type = {"f32": capi.TL_FLOAT32, "f16": capi.TL_FLOAT16, "bf16": capi.TL_BFLOAT16}
    layout = {"half": capi.TL_ROTARY_HALF, "interleaved": capi.TL_ROTARY_INTERLEAVED}
    dev = s["q"].device

    def turn(d):
        spec = capi.TlRotarySpec(base=BASE, factor=FACTOR, original_length=ORIGINAL, dim=case["rotary"], scaling={
            "plain": capi.TL_ROTARY_PLAIN, "linear": capi.TL_ROTARY_LINEAR, "ntk": capi.TL_ROTARY_NTK,
            "parts": capi.TL_ROTARY_PARTS, "smooth": capi.TL_ROTARY_SMOOTH}[case["scaling"]])
        spec.low, spec.high = (1.0, 32.0) if case["scaling"] == "parts" else (1.0, 4.0)
        table, magnitude = (ctypes.c_uint64 * (case["rotary"] // 2))(), ctypes.c_float()
        capi.check(lib.tl_rotary_frequencies(ctypes.byref(spec), table, ctypes.byref(magnitude)), lib, "frequencies")
        s["frequencies"] = torch.frombuffer(bytearray(table), dtype=torch.int64).to(dev)
        d.frequencies, d.magnitude = s["frequencies"].data_ptr(), magnitude.value
        d.rotary_dim, d.layout, d.norm, d.eps = case["rotary"], layout[case["layout"]], int(case["norm"]), EPS

    def view(x):  # [B, T, H, D] or [tokens, H, D]
        b = x.stride(0) if x.dim() == 4 else 0
        return capi.TlHeadView(x.data_ptr(), b, x.stride(-2), x.stride(-3))

    if case["kind"] in ("rotate", "rotate_grad"):
        d = capi.TlRotaryDesc(B=case["batch"], T=case["tokens"], D=case["dim"], type=type[case["type"]],
                              out_type=type[case["type"]])
        turn(d)
        d.positions = s["positions"].data_ptr() if s["positions"] is not None else None
        for part, name in ((d.q, "q"), (d.k, "k")):
            part.heads, part.x = case[{"q": "q_heads", "k": "kv_heads"}[name]], view(s[name])
            if case["norm"]:
                part.weight = s[name + "_weight"].data_ptr()
            if case["kind"] == "rotate":
                part.out = view(s[name + "_out"])
            else:
                part.d_out, part.dx = view(s[f"d{name}_out"]), view(s["d" + name])
                if case["norm"]:
                    part.dweight = s[f"d{name}_weight"].data_ptr()
        call = lib.tl_rotary_heads if case["kind"] == "rotate" else lib.tl_rotary_heads_backward
        size = lib.tl_rotary_heads_workspace_size
    else:
        d = capi.TlCacheAppendDesc() if case["kind"] == "append" else capi.TlPagedAttentionDesc()
        c, k = d.cache, s["k_cache"]
        c.k, c.v = k.data_ptr(), s["v_cache"].data_ptr()
        c.page_stride, c.slot_stride, c.head_stride = k.stride(0), k.stride(1), k.stride(2)
        c.pages, c.page_size, c.heads, c.D = k.shape
        c.type = type[case["type"]]
        c.table, c.table_stride, c.sequences = s["table"].data_ptr(), s["table"].stride(0), case["sequences"]
        c.starts, c.lengths, c.tokens = s["starts"].data_ptr(), s["keys"].data_ptr(), s["q"].shape[0]
        d.q, d.q_heads = view(s["q"]), case["q_heads"]
        if case["kind"] == "append":
            turn(d)
            d.k, d.v, d.q_out, d.type = view(s["k"]), view(s["v"]), view(s["q_out"]), type[case["from"]]
            d.q_out_type = type[case["type"]]
            if case["norm"]:
                d.q_weight, d.k_weight = s["q_weight"].data_ptr(), s["k_weight"].data_ptr()
            call, size = lib.tl_cache_append, None
        else:
            d.out, d.lse, d.out_type = view(s["out"]), s["lse"].data_ptr(), type[case["type"]]
            d.scale, d.causal, d.window = 1.0 / math.sqrt(case["dim"]), 1, case["window"]
            # what the program knows of the batch's lengths without reading them back
            d.max_length, d.max_new = case["keys"], case["new"]
            call, size = lib.tl_paged_attention, lib.tl_paged_attention_workspace_size
    if size:
        bytes = size(ctypes.byref(d))
        s["workspace"] = torch.empty(max(bytes, 1), dtype=torch.uint8, device=dev)
        d.workspace, d.workspace_bytes = s["workspace"].data_ptr(), bytes
    return call, (ctypes.byref(d), capi.check, lib)


OUTPUTS = {"rotate": ("q_out", "k_out"), "rotate_grad": ("dq", "dk", "dq_weight", "dk_weight"),
           "append": ("q_out", "k_cache", "v_cache"), "attend": ("out", "lse")}
PLAIN = {"rotate": _rotate_plain, "rotate_grad": _rotate_grad_plain, "append": _append_plain, "attend": _attend_plain}


def run(state):
    kind = state["case"]["kind"]
    if not own:
        out = PLAIN[kind](state)
        return {name: out[name] for name in OUTPUTS[kind] if name in out}
    ref, check, lib = state["plan"]
    rc = state["call"](ref, torch.cuda.current_stream().cuda_stream)
    if rc:
        check(rc, lib, kind)
    return {name: state[name] for name in OUTPUTS[kind] if name in state}


# ----------------------------------------------------------------- 64 bits

def exact(case, seed):
    """Every output from its definition in 64 bits, written with complex numbers and whole softmaxes."""
    s = prepare(case, seed)
    if case["kind"] == "attend":
        return _exact_attention(s) if work(case)["flops"] < 4e12 else None
    if case["kind"] == "append":
        at = _new_positions(s)
        q, k = (_exact_heads(s, n, at, _exact_norm(s, n, s[n].double())[0]) for n in ("q", "k"))
        k_cache, v_cache = s["k_cache"].double(), s["v_cache"].double()
        for i, (new, keys) in enumerate(s["lengths"]):
            for a in range(keys - new, keys):
                n = s["starts_host"][i] + a - (keys - new)
                where = (s["table"][i, a // case["page"]].long(), a % case["page"])
                k_cache[where], v_cache[where] = k[n], s["v"][n].double()
        return {"q_out": q, "k_cache": k_cache, "v_cache": v_cache}
    at, out = _heads_positions(s), {}
    for n in ("q", "k"):
        y, x, rms = _exact_norm(s, n, s[n].double())
        if case["kind"] == "rotate":
            out[n + "_out"] = _exact_heads(s, n, at, y)
            continue
        g = _exact_heads(s, n, -at.double(), s[f"d{n}_out"].double())
        if case["norm"]:
            out[f"d{n}_weight"] = (g * x).flatten(0, 2).sum(0)
            g = g * s[n + "_weight"].double()
            g = (g - x * (g * x).sum(-1, keepdim=True) / case["dim"]) / rms
        out["d" + n] = g
    return {name: out[name] for name in OUTPUTS[case["kind"]] if name in out}


def _exact_norm(s, name, x):
    if not s["case"]["norm"]:
        return x, x, None
    rms = (x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt()
    return x / rms * s[name + "_weight"].double(), x / rms, rms


def _exact_heads(s, name, at, x):
    case, r = s["case"], s["case"]["rotary"]
    turned, rest = x[..., :r], x[..., r:]
    pairs = turned.unflatten(-1, (2, r // 2)).transpose(-1, -2) if case["layout"] == "half" else turned.unflatten(-1, (r // 2, 2))
    phase = at.double()[..., None, None] * s["radians"]
    z = torch.view_as_complex(pairs.contiguous()) * torch.polar(torch.full_like(phase, s["magnitude"]), phase)
    z = torch.view_as_real(z)
    z = z.transpose(-1, -2) if case["layout"] == "half" else z
    return torch.cat((z.flatten(-2), rest), -1)


def _exact_attention(s):
    case, outs, lses = s["case"], [], []
    group = case["q_heads"] // case["kv_heads"]
    for i, (new, keys) in enumerate(s["lengths"]):
        place = torch.arange(keys, device=s["q"].device)
        page, slot = s["table"][i].long()[place // case["page"]], place % case["page"]
        q = s["q"][s["starts_host"][i]:s["starts_host"][i + 1]]
        back = (place[keys - new:, None] - place[None, :])
        allowed = (back >= 0) & (back < (case["window"] or keys + 1))
        out, lse = [], []
        for head in range(case["q_heads"]):
            k, v = (s[c][page, slot, head // group].double() for c in ("k_cache", "v_cache"))
            x = (q[:, head].double() @ k.T / case["dim"] ** 0.5).where(allowed, torch.tensor(-math.inf, dtype=torch.float64, device=q.device))
            out.append(torch.softmax(x, 1) @ v)
            lse.append(torch.logsumexp(x, 1))
        outs.append(torch.stack(out, 1))
        lses.append(torch.stack(lse, 1))
    return {"out": torch.cat(outs), "lse": torch.cat(lses)}
