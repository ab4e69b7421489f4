"""Measured workloads of the token scoring and distillation operators.

Five entry points of include/templit_cuda.h, over rows of next-token logits:

  score          tl_token_logprob_rows: log probability of a given token, entropy, top alternatives
  score_grad     tl_token_logprob_backward_rows: the gradient of both towards the logits
  distill        tl_distill_rows: loss of a student against a teacher's top tokens (and hard targets)
  distill_grad   tl_distill_backward_rows: its gradient, from the statistics the forward kept
  distill_train  tl_distill_train_rows: loss and gradient in one call

`own` chooses between the plain form (elementary torch operations in 32 bits) and the kernels.
Vocabulary 2048 and 12288 = 64 x 192 rows are the framework's own training step; the long
vocabularies are generic.
"""
import ctypes
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
KINDS = ("score", "score_grad", "distill", "distill_grad", "distill_train")
STATS = 8       # floats per row that the distillation forward keeps for the backward
NO_TOKEN = -1   # 0xffffffff: a row without a given token
LARGEST = 4096 * 128000  # elements of the largest listed case
LOSS_SCALE = {"f32": 1.0, "f16": 1024.0, "bf16": 1.0}  # keeps 16-bit gradients in float16's range


def _case(name, kind, rows, vocab, type, top, **more):
    c = {"name": name, "kind": kind, "rows": rows, "vocab": vocab, "type": type, "top": top,
         "pad": 0, "temperature": 1.0, "masked": False, "tail": False, "hard": False}
    c.update(more)
    return c


def listed():
    return [
        # one generated token of the framework's own model: log probability and five alternatives
        _case("score_one_token", "score", 1, 2048, "f32", 5),
        # one decoding step of 64 sequences, long odd vocabulary, a third of it not allowed
        _case("score_decode_64", "score", 64, 50001, "bf16", 20, temperature=0.7, masked=True),
        # the teacher's side of the framework's training batch: 64 sequences of 192 tokens
        _case("score_teacher_batch", "score", 12288, 2048, "f32", 32, temperature=2.0),
        # scoring a corpus under a long vocabulary
        _case("score_corpus", "score", 4096, 128000, "bf16", 20),
        # policy gradient with an entropy bonus, the framework's training batch
        _case("score_grad_batch", "score_grad", 12288, 2048, "f32", 0),
        # the same, long odd vocabulary (no row but the first is 16-byte aligned)
        _case("score_grad_odd", "score_grad", 4096, 50001, "bf16", 0, temperature=0.9),
        # validation of a student on one sequence
        _case("distill_one_sequence", "distill", 192, 2048, "f32", 16, temperature=2.0, hard=True),
        # validation on a large batch, long vocabulary, with the teacher's remaining mass
        _case("distill_corpus", "distill", 4096, 128000, "bf16", 64, tail=True),
        # the backward pass alone, framework's batch
        _case("distill_grad_batch", "distill_grad", 12288, 2048, "f32", 32, temperature=2.0, tail=True, hard=True),
        # the backward pass alone, long vocabulary in padded rows
        _case("distill_grad_padded", "distill_grad", 4096, 65501, "f16", 64, temperature=1.5, pad=35),
        # one training step's loss and gradient, framework's batch
        _case("distill_train_batch", "distill_train", 12288, 2048, "f32", 32, temperature=2.0, tail=True, hard=True),
        # one training step's loss and gradient, long vocabulary
        _case("distill_train_corpus", "distill_train", 4096, 128000, "bf16", 64, tail=True),
    ]


def draw(rng):
    spread = lambda a, b: int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))  # noqa: E731
    kind = rng.choice(KINDS)
    vocab = spread(200, 200000)
    rows = max(1, min(spread(1, 16384), LARGEST // vocab))
    type = rng.choice(("f32", "f16", "bf16"))
    if type == "f32":
        rows = max(1, min(rows, LARGEST // (2 * vocab)))
    distil = kind.startswith("distill")
    top = 0 if kind == "score_grad" else rng.randint(1, 128) if distil else rng.choice((0, 1, rng.randint(2, 40), rng.randint(2, 128)))
    return {"kind": kind, "rows": rows, "vocab": vocab, "type": type, "top": top,
            "pad": rng.choice((0, 0, rng.randint(1, 64))), "temperature": round(rng.uniform(0.5, 4.0), 2) if rng.random() < 0.6 else 1.0,
            "masked": not distil and rng.random() < 0.3, "tail": distil and rng.random() < 0.5, "hard": distil and rng.random() < 0.5}


def work(case):
    n, v, b, k = case["rows"], case["vocab"], BYTES[case["type"]], case["top"]
    grads = case["kind"] in ("score_grad", "distill_grad", "distill_train")
    per_row = {"score": 4 + 16 + 8 * k, "score_grad": 24, "distill": 8 * k + 8 + 4 * STATS,
               "distill_grad": 8 * k + 4 + 4 * STATS, "distill_train": 8 * k + 12 + 4 * STATS}[case["kind"]]
    if case["hard"]:
        per_row += 4
    # a subtraction, an exponential and an addition per logit; the gradient another two operations
    return {"bytes": n * (v * b * (2 if grads else 1) + per_row), "flops": n * v * (5 if grads else 3)}


# ------------------------------------------------------------------ inputs

def _logits(case, gen, dev):
    """Next-token logits: a Zipf-like preference for some tokens, rows of different sharpness."""
    n, v = case["rows"], case["vocab"]
    order = torch.randperm(v, generator=gen, device=dev).float()
    favour = 6.0 - 1.1 * torch.log1p(order)
    sharp = 0.5 + 2.5 * torch.rand(n, 1, generator=gen, device=dev)
    return torch.randn(n, v, generator=gen, device=dev).mul_(sharp).add_(favour)


def _rows(case, dev):
    """A [rows, vocab] view whose rows lie vocab + pad elements apart."""
    return torch.zeros(case["rows"], case["vocab"] + case["pad"], dtype=TYPES[case["type"]], device=dev)[:, :case["vocab"]]


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    n, v, k, tau = case["rows"], case["vocab"], min(case["top"], case["vocab"]), case["temperature"]
    s = {"case": case, "kind": case["kind"], "tau": tau, "k": k}
    mean = LOSS_SCALE[case["type"]] / n
    z = _logits(case, gen, dev)
    s["logits"] = _rows(case, dev)
    # tokens that the model itself finds likely: the second of a few drawn ones
    some = torch.randint(0, v, (n, 8), generator=gen, device=dev)
    targets = some.gather(1, z.gather(1, some).argmax(1, keepdim=True))[:, 0]
    if case["masked"]:
        shut = torch.rand(v, generator=gen, device=dev) < 0.33
        shut[targets] = False
        z.masked_fill_(shut, -math.inf)
    s["targets"] = targets.to(torch.int32)
    floats = lambda *shape: torch.empty(shape, device=dev)  # noqa: E731
    if s["kind"].startswith("distill"):
        # the teacher's top log probabilities at the distillation temperature, as scoring gives them
        values, ids = z.topk(k, dim=1)
        s["teacher"] = (values / tau - torch.logsumexp(z / tau, 1, keepdim=True)).contiguous()
        s["teacher_ids"] = ids.to(torch.int32).contiguous()
        s["kd"], s["ce"] = (0.9 * tau * tau, 0.1) if case["hard"] else (tau * tau, 0.0)
        s["scale"] = torch.full((n,), mean, device=dev)
        z.mul_(0.8).add_(torch.randn(n, v, generator=gen, device=dev), alpha=0.7)  # the student
        s["logits"].copy_(z)
        s["loss"], s["kl"], s["stats"] = floats(n), floats(n), floats(n, STATS)
        if s["kind"] == "distill_grad":
            s["stats"].copy_(_distill_plain(s)["stats"])
    else:
        s["logits"].copy_(z)
        s["logprob"], s["entropy"], s["stats"] = floats(n), floats(n), floats(n, 2)
        s["top_logprob"] = floats(n, k)
        s["top_ids"] = torch.empty(n, k, dtype=torch.int32, device=dev)
        if s["kind"] == "score_grad":
            del z
            kept = _score_plain(s)
            s["stats"].copy_(kept["stats"])
            s["entropy"].copy_(kept["entropy"])
            s["d_logprob"] = torch.randn(n, generator=gen, device=dev) * mean  # advantages
            s["d_entropy"] = torch.full((n,), 0.01 * mean, device=dev)
    if s["kind"] in ("score_grad", "distill_grad", "distill_train"):
        s["dlogits"] = _rows(case, dev)
    if own:
        s["call"], s["plan"] = _plan(s)
    return s


# --------------------------------------------------------------- plain form

def _order(z):
    """Whole numbers that order the logits, the lower index first among equals."""
    bits = (z.float() + 0.0).view(torch.int32)
    bits = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
    last = z.shape[1] - 1
    return bits * (1 << 32) + (last - torch.arange(z.shape[1], device=z.device))


def _score_plain(s):
    z, tau, k = s["logits"].float(), s["tau"], s["k"]
    m = z.max(1, keepdim=True).values
    x = (z - m) / tau
    e = x.exp()
    total = e.sum(1, keepdim=True)
    log_total = total.log()
    out = {"logprob": x.gather(1, s["targets"].long()[:, None])[:, 0] - log_total[:, 0],
           "entropy": log_total[:, 0] - (e * x.clamp_min(-1e4)).sum(1) / total[:, 0],
           "stats": torch.cat((m, total), 1)}
    if k:
        last = z.shape[1] - 1
        ids = last - (_order(s["logits"]).topk(k, dim=1).values & 0xFFFFFFFF)
        out["top_ids"] = ids.to(torch.int32)
        out["top_logprob"] = x.gather(1, ids) - log_total
    return out


def _score_grad_plain(s):
    z, tau = s["logits"].float(), s["tau"]
    m, total = s["stats"][:, :1], s["stats"][:, 1:]
    x = (z - m) / tau
    q = x.exp() / total
    g = -s["d_logprob"][:, None] * q
    g -= s["d_entropy"][:, None] * q * (x.clamp_min(-1e4) - total.log() + s["entropy"][:, None])
    g.scatter_add_(1, s["targets"].long()[:, None], s["d_logprob"][:, None])
    return {"dlogits": (g / tau).to(s["logits"].dtype)}


def _teacher_plain(s):
    u = s["teacher"]
    if s["case"]["tail"]:
        p = u.exp()
        shift, unit = torch.zeros_like(u[:, :1]), torch.ones_like(u[:, :1])
        rest = (1.0 - p.sum(1, keepdim=True)).clamp_min(0.0)
    else:
        shift = u.max(1, keepdim=True).values
        unit = 1.0 / (u - shift).exp().sum(1, keepdim=True)
        p = (u - shift).exp() * unit
        rest = torch.zeros_like(shift)
    return p, rest, shift, unit


def _distill_plain(s):
    z, tau, ids = s["logits"].float(), s["tau"], s["teacher_ids"].long()
    p, rest, shift, unit = _teacher_plain(s)
    m = z.max(1, keepdim=True).values
    x = (z - m) / tau
    total = x.exp().sum(1, keepdim=True)
    first = (z - m).exp().sum(1, keepdim=True) if s["case"]["hard"] else torch.zeros_like(m)
    log_q = x.gather(1, ids) - total.log()
    kl = (p * (p.clamp_min(1e-38).log() - log_q)).sum(1)
    if s["case"]["tail"]:
        others = z.scatter(1, ids, -math.inf)
        m_rest = others.max(1, keepdim=True).values
        s_rest = ((others - m_rest) / tau).exp().sum(1, keepdim=True)
        log_rest = (m_rest - m) / tau + s_rest.log() - total.log()
        kl += (rest * (rest.clamp_min(1e-38).log() - log_rest))[:, 0]
        coef = (log_rest.exp() - rest) / s_rest
    else:
        m_rest, coef = m, 1.0 / total
    loss = s["kd"] * kl
    if s["case"]["hard"]:
        loss = loss - s["ce"] * ((z.gather(1, s["targets"].long()[:, None]) - m) - first.log())[:, 0]
    return {"loss": loss, "kl": kl,
            "stats": torch.cat((m, total, first, m_rest, coef, shift, unit, torch.zeros_like(m)), 1)}


def _distill_grad_plain(s, stats):
    z, tau, ids = s["logits"].float(), s["tau"], s["teacher_ids"].long()
    m, total, first, m_rest, coef, shift, unit, _ = stats.split(1, 1)
    p = (s["teacher"] - shift).exp() * unit
    g = ((z - m_rest) / tau).exp() * coef
    g.scatter_(1, ids, ((z.gather(1, ids) - m) / tau).exp() / total - p)
    g *= s["kd"] / tau
    if s["case"]["hard"]:
        g += s["ce"] * ((z - m).exp() / first)
        g.scatter_add_(1, s["targets"].long()[:, None], torch.full_like(m, -s["ce"]))
    return {"dlogits": (g * s["scale"][:, None]).to(s["logits"].dtype)}


def _distill_train_plain(s):
    out = _distill_plain(s)
    return {**out, **_distill_grad_plain(s, out["stats"])}


# ------------------------------------------------------------------ kernels

def _plan(s):
    """The call and its descriptor: the pointers and sizes that a program fills in once."""
    from templit_b200 import capi
    lib, case, z = capi.cuda_lib(), s["case"], s["logits"]
    d = capi.TlDistillDesc() if s["kind"].startswith("distill") else capi.TlTokenLogprobDesc()
    d.logits, d.row_stride = z.data_ptr(), z.stride(0)
    d.type = {"f32": capi.TL_FLOAT32, "f16": capi.TL_FLOAT16, "bf16": capi.TL_BFLOAT16}[case["type"]]
    d.rows, d.vocab, d.top, d.temperature = case["rows"], case["vocab"], s["k"], s["tau"]
    d.stats = s["stats"].data_ptr()
    if "dlogits" in s:
        d.dlogits, d.d_row_stride = s["dlogits"].data_ptr(), s["dlogits"].stride(0)
    if s["kind"].startswith("distill"):
        d.teacher, d.teacher_ids, d.teacher_temperature = s["teacher"].data_ptr(), s["teacher_ids"].data_ptr(), 1.0
        d.tail = capi.TL_DISTILL_TAIL if case["tail"] else capi.TL_DISTILL_RENORM
        d.kd_weight, d.ce_weight = s["kd"], s["ce"]
        d.targets = s["targets"].data_ptr() if case["hard"] else None
        d.row_scale, d.loss, d.kl = s["scale"].data_ptr(), s["loss"].data_ptr(), s["kl"].data_ptr()
    else:
        d.targets, d.entropy = s["targets"].data_ptr(), s["entropy"].data_ptr()
        if s["kind"] == "score":
            d.logprob = s["logprob"].data_ptr()
            if s["k"]:
                d.top_logprob, d.top_ids = s["top_logprob"].data_ptr(), s["top_ids"].data_ptr()
        else:
            d.d_logprob, d.d_entropy = s["d_logprob"].data_ptr(), s["d_entropy"].data_ptr()
    call = {"score": lib.tl_token_logprob_rows, "score_grad": lib.tl_token_logprob_backward_rows,
            "distill": lib.tl_distill_rows, "distill_grad": lib.tl_distill_backward_rows,
            "distill_train": lib.tl_distill_train_rows}[s["kind"]]
    return call, (ctypes.byref(d), capi.check, lib)


OUTPUTS = {"score": ("logprob", "entropy", "stats", "top_logprob", "top_ids"), "score_grad": ("dlogits",),
           "distill": ("loss", "kl", "stats"), "distill_grad": ("dlogits",),
           "distill_train": ("loss", "kl", "stats", "dlogits")}
PLAIN = {"score": _score_plain, "score_grad": _score_grad_plain, "distill": _distill_plain,
         "distill_grad": lambda s: _distill_grad_plain(s, s["stats"]), "distill_train": _distill_train_plain}


def run(state):
    if not own:
        return PLAIN[state["kind"]](state)
    ref, check, lib = state["plan"]
    rc = state["call"](ref, torch.cuda.current_stream().cuda_stream)
    if rc:
        check(rc, lib, state["kind"])
    return {name: state[name] for name in OUTPUTS[state["kind"]] if not name.startswith("top_") or state["k"]}


# ----------------------------------------------------------------- 64 bits

def exact(case, seed):
    """Every output from its definition over whole rows in 64 bits, a few rows at a time."""
    s = prepare(case, seed)
    step = max(1, (1 << 27) // case["vocab"])
    parts = []
    for a in range(0, case["rows"], step):
        parts.append(_exact_rows(s, slice(a, min(case["rows"], a + step))))
    out = {name: torch.cat([p[name] for p in parts]) for name in parts[0]}
    for name in OUTPUTS[case["kind"]]:
        if name.startswith("top_") and not s["k"]:
            continue
        out.setdefault(name, None)
    return out


def _exact_rows(s, at):
    case, tau, k = s["case"], s["tau"], s["k"]
    z = s["logits"][at].double()
    log_q = torch.log_softmax(z / tau, 1)
    token = s["targets"][at].long()[:, None]
    here = torch.arange(z.shape[0], device=z.device)[:, None]
    if case["kind"] == "score":
        out = {"logprob": log_q[here, token][:, 0], "entropy": torch.special.entr(log_q.exp()).sum(1)}
        if k:
            out["top_logprob"] = log_q.topk(k, dim=1).values
        return out
    q = log_q.exp()
    if case["kind"] == "score_grad":
        a, b = s["d_logprob"][at].double()[:, None], s["d_entropy"][at].double()[:, None]
        inner = -torch.special.entr(q)           # q log q, 0 where q is
        g = -a * q - b * (inner - q * inner.sum(1, keepdim=True))
        g[here, token] += a
        return {"dlogits": g / tau}
    ids = s["teacher_ids"][at].long()
    u = s["teacher"][at].double()
    p = torch.zeros_like(q).scatter_(1, ids, u.exp() if case["tail"] else torch.softmax(u, 1))
    kl = (torch.special.xlogy(p, p) - p * log_q).sum(1)
    grad = q - p
    if case["tail"]:
        outside = torch.ones_like(q).scatter_(1, ids, 0.0)
        mass = (1.0 - p.sum(1, keepdim=True)).clamp_min(0.0)
        share = q * outside
        left = share.sum(1, keepdim=True)
        kl += (torch.special.xlogy(mass, mass) - mass * left.log())[:, 0]
        grad -= mass * share / left
    loss = s["kd"] * kl
    grad *= s["kd"] / tau
    if case["hard"]:
        log_1 = torch.log_softmax(z, 1)
        loss = loss - s["ce"] * log_1[here, token][:, 0]
        grad += s["ce"] * log_1.exp()
        grad[here, token] -= s["ce"]
    out = {}
    if case["kind"] != "distill_grad":
        out.update(loss=loss, kl=kl)
    if case["kind"] != "distill":
        out["dlogits"] = grad * s["scale"][at].double()[:, None]
    return out
