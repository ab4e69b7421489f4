"""The token scoring and distillation entry points without a GPU: the
descriptors' layout in ctypes against the C compiler's, and every refusal,
which comes before any device call."""
import ctypes
import math
import os
import shutil
import subprocess

import pytest

from templit_b200 import capi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.skipif(not shutil.which("gcc"), reason="no C compiler for the layout check")
def test_descriptor_layouts(tmp_path):
    structs = {"tl_token_logprob_desc": capi.TlTokenLogprobDesc, "tl_distill_desc": capi.TlDistillDesc}
    lines = ["#include <stddef.h>", "#include <stdio.h>", '#include "templit_cuda.h"', "int main(void) {"]
    for name, py in structs.items():
        lines.append(f'  printf("{name} size %zu\\n", sizeof({name}));')
        lines += [f'  printf("{name} {f} %zu\\n", offsetof({name}, {f}));' for f, _ in py._fields_]
    lines += ['  printf("constants %u %u %u\\n", TL_TOKEN_MAX_TOP, TL_DISTILL_STATS, TL_DISTILL_MAX_VOCAB);',
              "  return 0;\n}"]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines))
    subprocess.run(["gcc", f"-I{ROOT}/include", str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines()
    assert out.pop() == f"constants {capi.TL_TOKEN_MAX_TOP} {capi.TL_DISTILL_STATS} {capi.TL_DISTILL_MAX_VOCAB}"
    got = dict(line.rsplit(" ", 1) for line in out)
    for name, py in structs.items():
        assert int(got[f"{name} size"]) == ctypes.sizeof(py)
        for f, _ in py._fields_:
            assert int(got[f"{name} {f}"]) == getattr(py, f).offset, (name, f)


SOME = 0x10000  # an address that a refused call never reads


def score_desc(**fields):
    d = capi.TlTokenLogprobDesc(logits=SOME, rows=4, vocab=16, top=2, temperature=1.0, targets=SOME,
                                logprob=SOME, entropy=SOME, stats=SOME, top_logprob=SOME,
                                top_ids=SOME, d_logprob=SOME, d_entropy=SOME, dlogits=2 * SOME)
    for k, v in fields.items():
        setattr(d, k, v)
    return d


def distill_desc(**fields):
    d = capi.TlDistillDesc(logits=SOME, rows=4, vocab=16, top=2, temperature=1.0,
                           teacher_temperature=1.0, kd_weight=1.0, ce_weight=0.5, teacher_ids=SOME,
                           teacher=SOME, targets=SOME, loss=SOME, stats=SOME, dlogits=2 * SOME)
    for k, v in fields.items():
        setattr(d, k, v)
    return d


def refused(name, desc, code, word):
    lib = capi.cuda_lib()
    rc = getattr(lib, name)(None if desc is None else ctypes.byref(desc), None)
    assert rc == code, (rc, lib.tl_last_error())
    assert name.encode() in lib.tl_last_error() and word in lib.tl_last_error(), lib.tl_last_error()


COMMON = [
    (dict(type=3), capi.TL_ERR_INVALID, b"type"),
    (dict(vocab=0, top=0), capi.TL_ERR_INVALID, b"final dimension"),
    (dict(vocab=(1 << 31) + 1), capi.TL_ERR_RANGE, b"2^31"),
    (dict(temperature=0.0), capi.TL_ERR_INVALID, b"temperature"),
    (dict(temperature=-1.0), capi.TL_ERR_INVALID, b"temperature"),
    (dict(temperature=math.inf), capi.TL_ERR_INVALID, b"temperature"),
    (dict(temperature=math.nan), capi.TL_ERR_INVALID, b"temperature"),
    (dict(row_stride=15), capi.TL_ERR_INVALID, b"stride"),
    (dict(row_stride=1 << 62), capi.TL_ERR_RANGE, b"address space"),
    (dict(logits=None), capi.TL_ERR_INVALID, b"null logits"),
    (dict(logits=SOME + 2), capi.TL_ERR_INVALID, b"aligned"),
    (dict(logits=SOME + 1, type=capi.TL_BFLOAT16), capi.TL_ERR_INVALID, b"aligned"),
]
GRADIENT = [
    (dict(dlogits=None), capi.TL_ERR_INVALID, b"null dlogits"),
    (dict(dlogits=SOME + 1), capi.TL_ERR_INVALID, b"aligned"),
    (dict(d_row_stride=15), capi.TL_ERR_INVALID, b"stride"),
    (dict(d_row_stride=1 << 62), capi.TL_ERR_RANGE, b"address space"),
    (dict(dlogits=SOME, row_stride=20), capi.TL_ERR_INVALID, b"in place"),
    (dict(stats=None), capi.TL_ERR_INVALID, b"null stats"),
]


@pytest.mark.parametrize("fields,code,word", COMMON + [
    (dict(top=17), capi.TL_ERR_INVALID, b"more alternatives"),
    (dict(top=129, vocab=200), capi.TL_ERR_RANGE, b"128"),
    (dict(targets=None), capi.TL_ERR_INVALID, b"together"),
    (dict(logprob=None), capi.TL_ERR_INVALID, b"together"),
    (dict(top_ids=None), capi.TL_ERR_INVALID, b"top_ids"),
    (dict(top_logprob=None), capi.TL_ERR_INVALID, b"top_logprob"),
    (dict(targets=None, logprob=None, entropy=None, stats=None, top=0), capi.TL_ERR_INVALID, b"no output"),
])
def test_scoring_refusals(fields, code, word):
    refused("tl_token_logprob_rows", score_desc(**fields), code, word)


@pytest.mark.parametrize("fields,code,word", COMMON + GRADIENT + [
    (dict(d_logprob=None, d_entropy=None), capi.TL_ERR_INVALID, b"no incoming"),
    (dict(targets=None), capi.TL_ERR_INVALID, b"targets"),
    (dict(entropy=None), capi.TL_ERR_INVALID, b"entropy"),
])
def test_scoring_gradient_refusals(fields, code, word):
    refused("tl_token_logprob_backward_rows", score_desc(**fields), code, word)


DISTILL = [c for c in COMMON if c[0] != dict(vocab=0, top=0)] + [
    (dict(vocab=0), capi.TL_ERR_INVALID, b"final dimension"),
    (dict(top=0), capi.TL_ERR_INVALID, b"no teacher slots"),
    (dict(top=17), capi.TL_ERR_INVALID, b"more teacher slots"),
    (dict(top=129, vocab=200), capi.TL_ERR_RANGE, b"128"),
    (dict(teacher_temperature=0.0), capi.TL_ERR_INVALID, b"teacher temperature"),
    (dict(kd_weight=math.nan), capi.TL_ERR_INVALID, b"weights"),
    (dict(ce_weight=math.inf), capi.TL_ERR_INVALID, b"weights"),
    (dict(tail=2), capi.TL_ERR_INVALID, b"tail"),
    (dict(tail=1, vocab=capi.TL_DISTILL_MAX_VOCAB + 1), capi.TL_ERR_RANGE, b"too long"),
    (dict(teacher=None), capi.TL_ERR_INVALID, b"teacher"),
    (dict(teacher_ids=None), capi.TL_ERR_INVALID, b"teacher"),
]


@pytest.mark.parametrize("fields,code,word", DISTILL + [(dict(loss=None), capi.TL_ERR_INVALID, b"loss")])
def test_distillation_refusals(fields, code, word):
    refused("tl_distill_rows", distill_desc(**fields), code, word)


@pytest.mark.parametrize("fields,code,word",
                         DISTILL + GRADIENT[:-1] + [(dict(loss=None), capi.TL_ERR_INVALID, b"loss")])
def test_distillation_training_refusals(fields, code, word):
    refused("tl_distill_train_rows", distill_desc(**fields), code, word)


@pytest.mark.parametrize("fields,code,word", DISTILL + GRADIENT)
def test_distillation_gradient_refusals(fields, code, word):
    refused("tl_distill_backward_rows", distill_desc(**fields), code, word)


def test_null_descriptors_and_no_rows():
    lib = capi.cuda_lib()
    for name, desc in (("tl_token_logprob_rows", score_desc), ("tl_token_logprob_backward_rows", score_desc),
                       ("tl_distill_rows", distill_desc), ("tl_distill_backward_rows", distill_desc),
                       ("tl_distill_train_rows", distill_desc)):
        refused(name, None, capi.TL_ERR_INVALID, b"null descriptor")
        assert getattr(lib, name)(ctypes.byref(desc(rows=0, logits=None)), None) == capi.TL_OK
