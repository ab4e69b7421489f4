"""Temperatures whose reciprocal is beyond fp32: refused by every entry point
of token scoring and distillation, before any device call."""
import ctypes

import pytest

from templit_b200 import capi
from tests.test_token_rows_abi import distill_desc, refused, score_desc

SCORING = ["tl_token_logprob_rows", "tl_token_logprob_backward_rows"]
DISTILLATION = ["tl_distill_rows", "tl_distill_backward_rows", "tl_distill_train_rows"]


@pytest.mark.parametrize("temperature", [1e-45, 1e-40, 4.2e-39])
def test_refused(temperature):
    for name in SCORING:
        refused(name, score_desc(temperature=temperature), capi.TL_ERR_RANGE, b"temperature")
    for name in DISTILLATION:
        refused(name, distill_desc(temperature=temperature), capi.TL_ERR_RANGE, b"temperature")
    if temperature < 2.9e-39:  # 1 / temperature, without log2(e)
        for name in DISTILLATION:
            refused(name, distill_desc(teacher_temperature=temperature), capi.TL_ERR_RANGE, b"teacher temperature")


@pytest.mark.parametrize("temperature", [4.3e-39, 1e-38, 1e-3, 1.0, 3e38])
def test_taken(temperature):
    lib = capi.cuda_lib()
    for name in SCORING:
        assert getattr(lib, name)(ctypes.byref(score_desc(rows=0, temperature=temperature)), None) == capi.TL_OK
    for name in DISTILLATION:
        d = distill_desc(rows=0, temperature=temperature, teacher_temperature=temperature)
        assert getattr(lib, name)(ctypes.byref(d), None) == capi.TL_OK
