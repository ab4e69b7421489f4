"""More refusals of the rotation, cache and paged attention entry points,
without a GPU: what would fault there, or write a place twice."""
import ctypes

import pytest

from templit_b200 import capi
from tests.test_heads_abi import BAD, NOT, RANGE, SOME, append, attend, refused, rotary, view  # noqa: F401

WORK = dict(workspace=SOME, workspace_bytes=1 << 30)


@pytest.mark.parametrize("off", [1, 2, 3])
@pytest.mark.parametrize("name,make,fields,word", [
    ("tl_rotary_heads", rotary, dict(positions=SOME), b"positions"),
    ("tl_rotary_heads", rotary, dict(norm=1, q__weight=SOME), b"weight"),
    ("tl_rotary_heads_backward", rotary, dict(positions=SOME), b"positions"),
    ("tl_rotary_heads_backward", rotary, dict(norm=1, k__weight=SOME), b"weight"),
    ("tl_rotary_heads_backward", rotary, dict(norm=1, q__dweight=SOME, **WORK), b"dweight"),
    ("tl_cache_append", append, dict(norm=1, q_weight=SOME), b"weight"),
    ("tl_cache_append", append, dict(norm=1, k_weight=SOME), b"weight"),
    ("tl_cache_append", append, dict(cache__table=SOME), b"table"),
    ("tl_cache_append", append, dict(cache__starts=SOME), b"starts"),
    ("tl_cache_append", append, dict(cache__lengths=SOME), b"lengths"),
    ("tl_paged_attention", attend, dict(cache__table=SOME), b"table"),
    ("tl_paged_attention", attend, dict(cache__starts=SOME), b"starts"),
    ("tl_paged_attention", attend, dict(cache__lengths=SOME), b"lengths"),
    ("tl_paged_attention", attend, dict(lse=SOME), b"lse"),
])
def test_pointers_to_words_are_aligned(name, make, fields, word, off):
    *rest, last = [f for f in fields if f not in ("norm", *WORK)]
    refused(name, make(**{**fields, last: SOME + off}), BAD, word)


@pytest.mark.parametrize("apart", [0, 4, -252])
def test_weight_gradients_are_apart(apart):
    """Queries' and keys' are each set, not added to."""
    refused("tl_rotary_heads_backward", rotary(norm=1, q__dweight=SOME, k__dweight=SOME + apart, **WORK), BAD, b"dweight")


@pytest.mark.parametrize("name", ["tl_rotary_heads", "tl_rotary_heads_backward"])
@pytest.mark.parametrize("first,T", [((1 << 32) - 1, 2), ((1 << 32) - 2, 3), (1 << 31, (1 << 31) + 1)])
def test_positions_stay_in_32_bits(name, first, T):
    refused(name, rotary(first_position=first, T=T, B=1), RANGE, b"positions")


@pytest.mark.parametrize("scale", [2.4e38, -2.4e38, 3.4e38])
def test_scales_that_powers_of_two_cannot_hold(scale):
    refused("tl_paged_attention", attend(scale=scale), BAD, b"scale")


def test_very_long_sequences_are_not_waited_for():
    """Chunks of sequences that may have more than 2^26 keys go to the kernel without timed waits: its workspace."""
    lib = capi.cuda_lib()
    size = lambda **f: lib.tl_paged_attention_workspace_size(ctypes.byref(attend(  # noqa: E731
        cache__type=capi.TL_BFLOAT16, out_type=capi.TL_BFLOAT16, cache__tokens=64, cache__page_size=1 << 20, **f)))
    tiles, steps = size(cache__table_stride=64), size(cache__table_stride=64, max_new=1)
    assert tiles != steps
    assert size(cache__table_stride=65) == steps
    assert size(cache__table_stride=65, max_length=1 << 26) == tiles
    assert size(cache__table_stride=65, max_length=(1 << 26) + 1) == steps
