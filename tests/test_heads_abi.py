"""The rotation, cache and paged attention entry points without a GPU: the
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
    structs = {"tl_head_view": capi.TlHeadView, "tl_rotary_spec": capi.TlRotarySpec,
               "tl_rotary_part": capi.TlRotaryPart, "tl_rotary_desc": capi.TlRotaryDesc,
               "tl_paged_cache": capi.TlPagedCache, "tl_cache_append_desc": capi.TlCacheAppendDesc,
               "tl_paged_attention_desc": capi.TlPagedAttentionDesc}
    lines = ["#include <stddef.h>", "#include <stdio.h>", '#include "templit_cuda.h"', "int main(void) {"]
    for name, py in structs.items():
        lines.append(f'  printf("{name} size %zu\\n", sizeof({name}));')
        lines += [f'  printf("{name} {f} %zu\\n", offsetof({name}, {f}));' for f, _ in py._fields_]
    lines += ['  printf("constants %u %d %d\\n", TL_HEAD_MAX_DIM, TL_ROTARY_INTERLEAVED, TL_ROTARY_SMOOTH);',
              "  return 0;\n}"]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines))
    subprocess.run(["gcc", f"-I{ROOT}/include", str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines()
    assert out.pop() == f"constants {capi.TL_HEAD_MAX_DIM} {capi.TL_ROTARY_INTERLEAVED} {capi.TL_ROTARY_SMOOTH}"
    got = dict(line.rsplit(" ", 1) for line in out)
    for name, py in structs.items():
        assert int(got[f"{name} size"]) == ctypes.sizeof(py)
        for f, _ in py._fields_:
            assert int(got[f"{name} {f}"]) == getattr(py, f).offset, (name, f)


SOME = 0x10000  # an address that a refused call never reads


def view(p=SOME, b=0, h=64, r=256):
    return capi.TlHeadView(p, b, h, r)


def rotary(**fields):
    d = capi.TlRotaryDesc(B=2, T=3, D=64, rotary_dim=64, magnitude=1.0, eps=1e-6, frequencies=SOME)
    for part in (d.q, d.k):
        part.heads = 2
        part.x, part.d_out = view(b=768), view(2 * SOME, b=768)
        part.out, part.dx = view(3 * SOME, b=768), view(4 * SOME, b=768)
    for k, v in fields.items():
        at = d
        *path, last = k.split("__")
        for p in path:
            at = getattr(at, p)
        setattr(at, last, v)
    return d


def cache(c):
    c.k, c.v, c.pages, c.page_size, c.heads, c.D = SOME, 2 * SOME, 4, 16, 2, 64
    c.sequences, c.tokens, c.table_stride = 2, 5, 2
    c.table, c.lengths, c.starts = SOME, SOME, SOME


def append(**fields):
    d = capi.TlCacheAppendDesc(q=view(), k=view(), v=view(), q_out=view(2 * SOME), q_heads=4, rotary_dim=64,
                               magnitude=1.0, frequencies=SOME)
    cache(d.cache)
    return put(d, fields)


def attend(**fields):
    d = capi.TlPagedAttentionDesc(q=view(), out=view(2 * SOME), q_heads=4, scale=0.125, causal=1,
                                  workspace=SOME, workspace_bytes=1 << 40)
    cache(d.cache)
    return put(d, fields)


def put(d, fields):
    for k, v in fields.items():
        at = d
        *path, last = k.split("__")
        for p in path:
            at = getattr(at, p)
        setattr(at, last, v)
    return d


def refused(name, desc, code, word):
    lib = capi.cuda_lib()
    rc = getattr(lib, name)(None if desc is None else ctypes.byref(desc), None)
    assert rc == code, (rc, lib.tl_last_error())
    assert name.encode() in lib.tl_last_error() and word in lib.tl_last_error(), lib.tl_last_error()


BAD, RANGE, NOT = capi.TL_ERR_INVALID, capi.TL_ERR_RANGE, capi.TL_ERR_UNSUPPORTED
TURN = [
    (dict(layout=2), BAD, b"layout"), (dict(layout=-1), BAD, b"layout"), (dict(norm=2), BAD, b"norm"),
    (dict(norm=1, eps=-1.0), BAD, b"eps"), (dict(norm=1, eps=math.nan), BAD, b"eps"),
    (dict(norm=1, eps=math.inf), BAD, b"eps"), (dict(rotary_dim=63), BAD, b"rotary_dim"),
    (dict(rotary_dim=66), BAD, b"rotary_dim"), (dict(magnitude=math.nan), BAD, b"magnitude"),
    (dict(magnitude=math.inf), BAD, b"magnitude"), (dict(frequencies=None), BAD, b"frequencies"),
    (dict(frequencies=SOME + 4), BAD, b"frequencies"),
]
ROTARY = TURN + [
    (dict(type=3), BAD, b"type"), (dict(out_type=-1), BAD, b"type"),
    (dict(type=capi.TL_FLOAT16, out_type=capi.TL_BFLOAT16), NOT, b"fp16"),
    (dict(D=0, rotary_dim=0), RANGE, b"256"), (dict(D=257), RANGE, b"256"),
    (dict(B=1 << 20, T=1 << 13), RANGE, b"tokens"), (dict(q__heads=0, k__heads=0), BAD, b"heads"),
]


@pytest.mark.parametrize("fields,code,word", ROTARY + [
    (dict(q__x=view(None)), BAD, b"x is null"), (dict(k__out=view(None)), BAD, b"out is null"),
    (dict(q__x=view(SOME + 2)), BAD, b"aligned"), (dict(q__x=view(SOME + 1), type=1, out_type=1), BAD, b"aligned"),
    (dict(q__out=view(3 * SOME, 768, 63, 256)), BAD, b"stride"), (dict(q__out=view(3 * SOME, 768, 64, 0)), BAD, b"stride"),
    (dict(q__out=view(3 * SOME, 0, 64, 256)), BAD, b"stride"),
    (dict(q__x=view(SOME, 1 << 62, 64, 256)), RANGE, b"address"),
    (dict(q__out=view(SOME, 768, 64, 512)), BAD, b"out is x"), (dict(k__out=view(SOME, 768), out_type=1), BAD, b"out is x"),
])
def test_rotary_refusals(fields, code, word):
    refused("tl_rotary_heads", rotary(**fields), code, word)


@pytest.mark.parametrize("fields,code,word", ROTARY + [
    (dict(q__d_out=view(None)), BAD, b"d_out is null"), (dict(k__dx=view(None)), BAD, b"dx is null"),
    (dict(norm=1, q__x=view(None)), BAD, b"x is null"),
    (dict(q__dx=view(2 * SOME, 768, 64, 512)), BAD, b"in place"), (dict(q__dx=view(2 * SOME, 768), type=1), BAD, b"in place"),
    (dict(q__dweight=SOME, workspace=SOME, workspace_bytes=1 << 30), BAD, b"dweight"),
    (dict(norm=1, q__dweight=SOME), BAD, b"workspace"),
    (dict(norm=1, k__dweight=SOME, workspace=SOME, workspace_bytes=16), BAD, b"workspace"),
    (dict(norm=1, k__dweight=SOME, workspace=SOME + 2, workspace_bytes=1 << 30), BAD, b"workspace"),
])
def test_rotary_backward_refusals(fields, code, word):
    refused("tl_rotary_heads_backward", rotary(**fields), code, word)


CACHE = [
    (dict(cache__type=3), BAD, b"cache type"), (dict(cache__D=0, rotary_dim=0), RANGE, b"256"),
    (dict(cache__heads=0), BAD, b"key heads"), (dict(cache__page_size=0), BAD, b"pages"),
    (dict(cache__sequences=(1 << 30) + 1), RANGE, b"sequences"),
    (dict(cache__page_stride=64, cache__slot_stride=64, cache__head_stride=63), BAD, b"stride"),
    (dict(cache__page_stride=64, cache__slot_stride=0, cache__head_stride=64), BAD, b"stride"),
    (dict(cache__page_stride=1 << 61, cache__slot_stride=64, cache__head_stride=64), RANGE, b"address"),
    (dict(cache__starts=None), BAD, b"starts"), (dict(cache__lengths=None), BAD, b"lengths"),
    (dict(cache__table=None), BAD, b"table"), (dict(cache__k=None), BAD, b"null cache"),
    (dict(cache__v=None), BAD, b"null cache"), (dict(cache__k=SOME + 2), BAD, b"aligned"),
]


@pytest.mark.parametrize("fields,code,word", CACHE + TURN + [
    (dict(type=3), BAD, b"type"), (dict(q_out_type=3), BAD, b"type"), (dict(type=1, cache__type=2), NOT, b"fp16"),
    (dict(type=1, q_out_type=2, cache__type=1), NOT, b"fp16"), (dict(cache__D=257), RANGE, b"256"),
    (dict(q=view(None)), BAD, b"q is null"), (dict(k=view(None)), BAD, b"k is null"), (dict(v=view(None)), BAD, b"v is null"),
    (dict(q_out=view(None)), BAD, b"q_out is null"), (dict(q_out=view(SOME, 0, 64, 512)), BAD, b"q_out is q"),
    (dict(q_out=view(2 * SOME, 0, 32, 256)), BAD, b"stride"),
])
def test_append_refusals(fields, code, word):
    refused("tl_cache_append", append(**fields), code, word)


@pytest.mark.parametrize("fields,code,word", [c for c in CACHE if "rotary_dim" not in c[0]] + [
    (dict(cache__D=136), NOT, b"128"), (dict(cache__D=60), NOT, b"128"), (dict(q_heads=0), BAD, b"q_heads"),
    (dict(q_heads=3), BAD, b"q_heads"), (dict(out_type=1), BAD, b"out_type"),
    (dict(out_type=2, cache__type=1), BAD, b"out_type"), (dict(causal=2), BAD, b"causal"),
    (dict(causal=0, window=4), BAD, b"window"), (dict(scale=math.nan), BAD, b"scale"), (dict(scale=math.inf), BAD, b"scale"),
    (dict(q=view(None)), BAD, b"q is null"), (dict(out=view(None)), BAD, b"out is null"),
    (dict(out=view(SOME)), BAD, b"out is q"), (dict(out=view(2 * SOME, 0, 32, 256)), BAD, b"stride"),
    (dict(q=view(SOME + 8)), NOT, b"16-byte"), (dict(out=view(2 * SOME, 0, 66, 264)), NOT, b"16-byte"),
    (dict(cache__k=SOME + 4), NOT, b"16-byte"),
    (dict(cache__page_stride=4100, cache__slot_stride=130, cache__head_stride=65), NOT, b"16-byte"),
])
def test_attention_refusals(fields, code, word):
    refused("tl_paged_attention", attend(**fields), code, word)


def test_null_descriptors_and_sizes():
    for name in ("tl_rotary_heads", "tl_rotary_heads_backward", "tl_cache_append", "tl_paged_attention"):
        refused(name, None, BAD, b"null descriptor")
    lib = capi.cuda_lib()
    assert lib.tl_rotary_heads_workspace_size(None) == 0
    assert lib.tl_paged_attention_workspace_size(None) == 0
    assert lib.tl_rotary_heads_workspace_size(ctypes.byref(rotary(norm=1))) == 0
    assert lib.tl_rotary_heads_workspace_size(ctypes.byref(rotary(norm=1, q__dweight=SOME))) > 0


def test_nothing_to_do_is_no_error():
    lib = capi.cuda_lib()
    assert lib.tl_rotary_heads(ctypes.byref(rotary(T=0, q__x=view(None))), None) == capi.TL_OK
    assert lib.tl_rotary_heads_backward(ctypes.byref(rotary(B=0)), None) == capi.TL_OK
    for make, name in ((append, "tl_cache_append"), (attend, "tl_paged_attention")):
        for empty in (dict(cache__tokens=0), dict(cache__sequences=0)):
            assert getattr(lib, name)(ctypes.byref(make(**empty, q=view(None))), None) == capi.TL_OK
