"""Trains a small student head on a teacher's top tokens, with the kernels of
libtemplit_cuda.so only (torch allocates the device memory and owns the
stream):

  teacher logits   tl_gemm
  its top tokens   tl_token_logprob_rows   once per batch, at the temperature
  per step         tl_gemm                 student logits = features W
                   tl_distill_train_rows   loss, and the gradient in place of
                                           the logits
                   tl_gemm                 dW = features^T dlogits
                   tl_multi_clip_adamw     clipped AdamW
  policy steps     tl_token_logprob_rows, tl_token_logprob_backward_rows
                                           raise the given tokens' log
                                           probability, with an entropy bonus
  at the end       tl_token_logprob_rows   the targets' log probability and
                                           the entropy of both models

Sizes are the 4-block model's head: vocabulary 2048, width 384, sequences of
192 tokens.  Usage: python examples/distill.py [steps]
"""
import ctypes
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from templit_b200 import capi  # noqa: E402

VOCAB, WIDTH, SEQUENCES, LENGTH = 2048, 384, 16, 192
TOP, TEMPERATURE = 32, 2.0
LR, BETA1, BETA2, DECAY, CLIP = 3e-3, 0.9, 0.95, 0.1, 1.0


class Head:
    """A [WIDTH, VOCAB] projection with its AdamW state."""

    def __init__(self, lib, generator, std):
        self.lib = lib
        self.w = torch.randn(WIDTH, VOCAB, generator=generator, device="cuda") * std
        self.grad, self.m1, self.m2 = (torch.zeros_like(self.w) for _ in range(3))
        self.scalars = torch.tensor([BETA1, BETA2, 1 - LR * DECAY, LR], device="cuda")
        self.sqnorm = torch.zeros(1, device="cuda")
        self.chunks = -(-self.w.numel() // capi.TL_OPT_CHUNK)
        self.scratch = torch.empty(lib.tl_multi_clip_adamw_workspace_size(self.chunks), dtype=torch.uint8,
                                   device="cuda")
        self.gemm_scratch = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
        self.step_count = 0

    def _gemm(self, **fields):
        d = capi.TlGemmDesc(precision=capi.TL_GEMM_3XTF32, workspace=self.gemm_scratch.data_ptr(),
                            workspace_bytes=self.gemm_scratch.numel(), **fields)
        capi.check(self.lib.tl_gemm(ctypes.byref(d), stream()), self.lib, "tl_gemm")

    def logits(self, x, out):
        self._gemm(a=x.data_ptr(), b=self.w.data_ptr(), c=out.data_ptr(), m=x.shape[0], n=VOCAB, k=WIDTH)

    def step(self, x, dlogits):
        """w -= AdamW of x^T dlogits."""
        self._gemm(a=x.data_ptr(), b=dlogits.data_ptr(), c=self.grad.data_ptr(), m=WIDTH, n=VOCAB,
                   k=x.shape[0], trans_a=1)
        self.step_count += 1
        slot = capi.TlParamSlot(param=self.w.data_ptr(), out=self.w.data_ptr(), grad=self.grad.data_ptr(),
                                m1=self.m1.data_ptr(), m2=self.m2.data_ptr(), count=self.w.numel(),
                                chunk0=0, step=self.step_count)
        slots = torch.frombuffer(bytearray(slot), dtype=torch.uint8).cuda()
        self.sqnorm.zero_()
        p = self.scalars.data_ptr()
        capi.check(self.lib.tl_multi_clip_adamw(
            slots.data_ptr(), 1, self.chunks, self.sqnorm.data_ptr(), CLIP, p, p + 4, p + 8, p + 12, 1e-8,
            self.scratch.data_ptr(), self.scratch.numel(), stream()), self.lib, "tl_multi_clip_adamw")


def stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def call(lib, name, desc):
    capi.check(getattr(lib, name)(ctypes.byref(desc), stream()), lib, name)


def score(lib, logits, targets, top=0, temperature=1.0):
    """Log probability, entropy, statistics and alternatives of rows of logits."""
    rows = logits.shape[0]
    out = {"logprob": torch.empty(rows, device="cuda"), "entropy": torch.empty(rows, device="cuda"),
           "stats": torch.empty(rows, 2, device="cuda"), "top_logprob": torch.empty(rows, top, device="cuda"),
           "top_ids": torch.empty(rows, top, dtype=torch.int32, device="cuda")}
    call(lib, "tl_token_logprob_rows", capi.TlTokenLogprobDesc(
        logits=logits.data_ptr(), rows=rows, vocab=VOCAB, top=top, temperature=temperature,
        targets=targets.data_ptr(), **{k: v.data_ptr() for k, v in out.items()}))
    return out


def run(steps=60, policy_steps=10, report=print):
    lib = capi.cuda_lib()
    gen = torch.Generator(device="cuda").manual_seed(0)
    rows = SEQUENCES * LENGTH
    features = torch.randn(rows, WIDTH, generator=gen, device="cuda")
    teacher, student = Head(lib, gen, 0.08), Head(lib, gen, 0.02)
    logits, dlogits = (torch.empty(rows, VOCAB, device="cuda") for _ in range(2))
    # the text: the teacher's choice, with one token in ten drawn at random,
    # and the last tokens of every sequence padding
    teacher.logits(features, logits)
    targets = logits.argmax(1).to(torch.int32)
    noise = torch.rand(rows, generator=gen, device="cuda") < 0.1
    targets[noise] = torch.randint(0, VOCAB, (int(noise.sum()),), generator=gen, device="cuda", dtype=torch.int32)
    padding = (torch.arange(rows, device="cuda") % LENGTH) >= LENGTH - 5
    targets[padding] = -1  # TL_NO_TOKEN
    tops = score(lib, logits, targets, TOP, TEMPERATURE)
    teacher_score = score(lib, logits, targets)
    tokens = int((~padding).sum())
    scale = (~padding).float() / tokens
    loss, kl = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")

    history = []
    for step in range(steps):
        student.logits(features, logits)
        call(lib, "tl_distill_train_rows", capi.TlDistillDesc(
            logits=logits.data_ptr(), rows=rows, vocab=VOCAB, top=TOP, temperature=TEMPERATURE,
            teacher_temperature=1.0, kd_weight=0.9 * TEMPERATURE ** 2, ce_weight=0.1,
            tail=capi.TL_DISTILL_TAIL, teacher_ids=tops["top_ids"].data_ptr(),
            teacher=tops["top_logprob"].data_ptr(), targets=targets.data_ptr(), loss=loss.data_ptr(),
            kl=kl.data_ptr(), row_scale=scale.data_ptr(), dlogits=logits.data_ptr()))
        student.step(features, logits)
        history.append((float((loss * scale).sum()), float((kl * scale).sum())))
        if step % 10 == 0 or step == steps - 1:
            report(f"step {step:3d}  loss {history[-1][0]:.4f}  KL {history[-1][1]:.4f}")

    d_entropy = (0.01 * scale).neg()  # a step down the gradient: minus the bonus
    policy = []
    for _ in range(policy_steps):
        student.logits(features, logits)
        s = score(lib, logits, targets)
        policy.append(float((s["logprob"] * scale).sum()))
        minus = scale.neg()
        call(lib, "tl_token_logprob_backward_rows", capi.TlTokenLogprobDesc(
            logits=logits.data_ptr(), rows=rows, vocab=VOCAB, temperature=1.0, targets=targets.data_ptr(),
            entropy=s["entropy"].data_ptr(), stats=s["stats"].data_ptr(), d_logprob=minus.data_ptr(),
            d_entropy=d_entropy.data_ptr(), dlogits=dlogits.data_ptr()))
        student.step(features, dlogits)
    student.logits(features, logits)
    student_score = score(lib, logits, targets)
    mean = lambda t: float((t * scale).sum())  # noqa: E731
    policy.append(mean(student_score["logprob"]))
    report(f"targets' log probability: teacher {mean(teacher_score['logprob']):.4f}, student after distillation "
           f"{policy[0]:.4f}, after {policy_steps} policy steps {policy[-1]:.4f}")
    report(f"entropy: teacher {mean(teacher_score['entropy']):.4f}, student {mean(student_score['entropy']):.4f}")
    return {"history": history, "policy": policy}


if __name__ == "__main__":
    run(int(sys.argv[1]) if len(sys.argv) > 1 else 60)
