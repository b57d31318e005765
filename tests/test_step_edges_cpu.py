"""Refusals of the serving-step operators where arguments lie over one another
(CPU only, before any device work)."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")

from test_step_cpu import BAD, P  # noqa: E402

from woolly_b200 import _lib  # noqa: E402


@pytest.mark.parametrize("at,ldq,code", [
    (16, 256, BAD), (1024, 256, BAD), (-1024, 256, BAD), (0, 512, BAD), (1024, 512, BAD), (2 * 1024 - 16, 256, BAD),
])
def test_tree_attention_refuses_an_output_over_its_queries(at, ldq, code):
    a = dict(qt=0, q=P + 4096, ldq=ldq, ck=P, cv=P, pages=1, t=P, ld=2, max_pages=2, lengths=P, start=P, pos=P,
             mask=None, words=0, n=1, rows=2, heads=4, kvh=2, hd=64, window=0, scale=0.125, out=P + 4096 + at, ws=P,
             nb=1 << 40)
    assert _lib.lib().wl_tree_attention(*a.values(), None) == code
    assert b"overlaps" in _lib.lib().wl_last_error()


@pytest.mark.parametrize("at,ld,ldo", [
    (4, 16, 16), (-4, 16, 16), (36, 16, 16), (28, 16, 16), (64, 16, 16), (64 * 2 + 36, 16, 16), (64, 16, 32),
    (0, 16, 32), (40, 20, 21), (36, 20, 20), (44, 20, 20),
])
def test_process_logits_refuses_an_output_over_other_rows(at, ld, ldo):
    c = _lib.LogitContext()
    at += P + 1024
    assert _lib.lib().wl_process_logits(0, P + 1024, ld, 4, 10, P, C.byref(c), at, ldo, None) == BAD
    assert b"process_logits: " in _lib.lib().wl_last_error()
