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
