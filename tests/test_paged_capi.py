"""Refusals of the C entry points of rope and the paged cache. They happen before
any HIP call, so they need no GPU; every pointer is a made-up aligned address that
is never followed."""

import ctypes
import os
import re
import subprocess

import pytest

import flashattn_cuda
from paged_reference import Paged, Rows

LIB = ctypes.CDLL(os.path.join(os.path.dirname(flashattn_cuda.__file__), "libflashattn_hip.so"))
LIB.fa_last_error.restype = ctypes.c_char_p
LIB.fa_attend_paged_workspace_bytes.restype = ctypes.c_size_t
P, I, F, L = ctypes.c_void_p, ctypes.c_int, ctypes.c_float, ctypes.c_int64
ADDRESS = 1 << 20


GOOD = dict(k_pages=ADDRESS, v_pages=ADDRESS, page_table=ADDRESS, seq_lens=ADDRESS,
            cu_tokens=ADDRESS, dtype=0, batch=2, tokens=3, kv_heads=2, head_dim=64, page_size=16,
            num_pages=8, max_pages=4)
ROW = dict(data=ADDRESS, token_stride=256, head_stride=64)

LIB.fa_rope.argtypes = [P, P, P, P] + [I] * 5 + [L] * 4 + [I, I, F, I, P]
LIB.fa_append_paged.argtypes = [P, P, P, P, P, I, P, I, I, F, P]
LIB.fa_attend_paged.argtypes = [P, P, P, I, F, P, ctypes.c_size_t, P]


HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include",
                      "flashattn_hip", "paged.h")


def test_header_declares_what_the_library_exports():
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    names = sorted(set(re.findall(r"\b(fa_\w+)\s*\(", text)))
    assert names == ["fa_append_paged", "fa_attend_paged", "fa_attend_paged_workspace_bytes",
                     "fa_rope"]
    assert all(hasattr(LIB, n) for n in names)


def test_header_stands_alone_in_c_with_these_structures(tmp_path):
    source = tmp_path / "sizes.c"
    source.write_text(f'''#include "{HEADER}"
_Static_assert(sizeof(fa_paged) == {ctypes.sizeof(Paged)}, "fa_paged");
_Static_assert(sizeof(fa_rows) == {ctypes.sizeof(Rows)}, "fa_rows");
''')
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-fsyntax-only", str(source)], check=True)


def _refused(rc, message):
    assert rc == 1 and message in LIB.fa_last_error().decode(), LIB.fa_last_error()


BAD_CACHE = [
    (dict(k_pages=None), "non-NULL"), (dict(cu_tokens=None), "non-NULL"),
    (dict(v_pages=ADDRESS + 8), "16-byte aligned"), (dict(seq_lens=ADDRESS + 2), "4-byte aligned"),
    (dict(dtype=2), "unknown dtype"), (dict(batch=0), "> 0"), (dict(tokens=0), "> 0"),
    (dict(kv_heads=-1), "> 0"), (dict(num_pages=0), "> 0"), (dict(max_pages=0), "> 0"),
    (dict(head_dim=96), "head_dim"), (dict(page_size=8), "power of two"),
    (dict(page_size=48), "power of two"), (dict(page_size=2048), "power of two"),
    (dict(page_size=1024, max_pages=2 ** 20), "max_pages * page_size"),
    (dict(tokens=2 ** 24 + 1), "packed tokens"), (dict(batch=2 ** 16 + 1), "2^16 sequences"), (dict(kv_heads=8193), "K/V heads"),
]


@pytest.mark.parametrize("change,message", BAD_CACHE)
def test_bad_cache(change, message):
    cache, row = Paged(**{**GOOD, **change}), Rows(**ROW)
    c, r = ctypes.byref(cache), ctypes.byref(row)
    _refused(LIB.fa_attend_paged(c, r, ADDRESS, 4, 0.1, ADDRESS, 1 << 40, None), message)
    _refused(LIB.fa_append_paged(c, r, r, None, None, 0, None, 0, 0, 1.0, None), message)


def test_no_cache():
    _refused(LIB.fa_attend_paged(None, None, None, 4, 0.1, None, 0, None), "non-NULL")


@pytest.mark.parametrize("change,message", [
    (dict(data=None), "non-NULL"), (dict(data=ADDRESS + 4), "16-byte aligned"),
    (dict(token_stride=65), "multiples of 8"), (dict(head_stride=4), "multiples of 8")])
def test_bad_rows(change, message):
    cache, row, good = Paged(**GOOD), Rows(**{**ROW, **change}), Rows(**ROW)
    c, r, g = ctypes.byref(cache), ctypes.byref(row), ctypes.byref(good)
    _refused(LIB.fa_attend_paged(c, r, ADDRESS, 4, 0.1, ADDRESS, 1 << 40, None), message)
    _refused(LIB.fa_append_paged(c, r, g, None, None, 0, None, 0, 0, 1.0, None), message)
    _refused(LIB.fa_append_paged(c, g, r, None, None, 0, None, 0, 0, 1.0, None), message)
    _refused(LIB.fa_append_paged(c, g, g, r, ADDRESS, 4, ADDRESS, 64, 0, 1.0, None), message)


@pytest.mark.parametrize("heads,scale,message", [
    (3, 0.1, "divide"), (0, 0.1, "divide"), (258, 0.1, "128 query heads"),
    (4, float("nan"), "scale"), (4, 3e38, "scale")])
def test_bad_attention(heads, scale, message):
    cache, row = Paged(**GOOD), Rows(**ROW)
    _refused(LIB.fa_attend_paged(ctypes.byref(cache), ctypes.byref(row), ADDRESS, heads, scale,
                                 ADDRESS, 1 << 40, None), message)


def test_bad_attention_output():
    cache, row = Paged(**GOOD), Rows(**ROW)
    for out in (None, ADDRESS + 8):
        _refused(LIB.fa_attend_paged(ctypes.byref(cache), ctypes.byref(row), out, 4, 0.1, ADDRESS,
                                     1 << 40, None), "out must be")


@pytest.mark.parametrize("args", [(0, 4, 2, 64), (3, 4, 3, 64), (3, 4, 2, 32), (3, 258, 2, 64)])
def test_bad_workspace_query(args):
    assert LIB.fa_attend_paged_workspace_bytes(*args) == 0 and LIB.fa_last_error()


@pytest.mark.parametrize("q_out,heads,freq,rotary,factor,message", [
    (None, 4, ADDRESS, 64, 1.0, "q_out"), (ADDRESS + 8, 4, ADDRESS, 64, 1.0, "q_out"),
    (ADDRESS, 3, ADDRESS, 64, 1.0, "divide"), (ADDRESS, 4, None, 64, 1.0, "inv_freq"),
    (ADDRESS, 4, ADDRESS + 4, 64, 1.0, "inv_freq"), (ADDRESS, 4, ADDRESS, 24, 1.0, "rotary_dim"),
    (ADDRESS, 4, ADDRESS, 80, 1.0, "rotary_dim"), (ADDRESS, 4, ADDRESS, -16, 1.0, "rotary_dim"),
    (ADDRESS, 4, ADDRESS, 64, float("inf"), "factor")])
def test_bad_rotation_of_an_append(q_out, heads, freq, rotary, factor, message):
    cache, row = Paged(**GOOD), Rows(**ROW)
    r = ctypes.byref(row)
    _refused(LIB.fa_append_paged(ctypes.byref(cache), r, r, r, q_out, heads, freq, rotary, 0,
                                 factor, None), message)


ROPE = dict(x=ADDRESS, out=ADDRESS, positions=ADDRESS, inv_freq=ADDRESS, dtype=1, batch=2, heads=3,
            seq=5, head_dim=64, xb=960, xh=320, xr=64, pb=5, rotary=64, interleaved=0, factor=1.0,
            backward=0, stream=None)


@pytest.mark.parametrize("change,message", [
    (dict(x=None), "non-NULL"), (dict(out=None), "non-NULL"), (dict(positions=None), "non-NULL"),
    (dict(inv_freq=None), "inv_freq"), (dict(x=ADDRESS + 2), "16-byte"),
    (dict(out=ADDRESS + 8), "16-byte"), (dict(xr=60), "multiples of 8"),
    (dict(positions=ADDRESS + 1), "4-byte"), (dict(dtype=7), "dtype"), (dict(head_dim=80), "head_dim"),
    (dict(rotary=72), "rotary_dim"), (dict(rotary=0), "rotary_dim"), (dict(batch=0), "> 0"),
    (dict(heads=0), "> 0"), (dict(seq=-1), "> 0"), (dict(heads=65536), "too large"),
    (dict(batch=2 ** 20, seq=2 ** 20), "too large"), (dict(factor=float("nan")), "factor")])
def test_bad_rope(change, message):
    _refused(LIB.fa_rope(*{**ROPE, **change}.values()), message)
