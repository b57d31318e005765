"""Refusals of the serving-step operators, before any device work (CPU only)."""
import ctypes as C

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from woolly_b200 import _lib, ops

BAD, UNS, SMALL, OK = (_lib.WL_ERR_INVALID_ARGUMENT, _lib.WL_ERR_UNSUPPORTED,
                       _lib.WL_ERR_BUFFER_TOO_SMALL, _lib.WL_OK)
_buf = np.zeros(4096 + 64, np.uint8)
P = (_buf.ctypes.data + 63) // 64 * 64  # host memory: a call that passed its checks would not read it here
ODD = P + 8


def tables(**kw):
    a = dict(t=P, ld=4, pages=4, lengths=P, counts=P + 256, n=2, free=P, cap=4, count=P, rows=8, parents=None,
             words=0, out={})
    a.update(kw)
    o = dict(row_start=P, requests=P, positions=P, slots=P, lengths=P + 512, status=P, free_count=P,
             page_start=P, mask=P)
    o.update(a["out"])
    return _lib.lib().wl_block_tables(a["t"], a["ld"], a["pages"], a["lengths"], a["counts"], a["n"], a["free"],
                                      a["cap"], a["count"], a["rows"], a["parents"], a["words"],
                                      C.byref(_lib.StepPlan(**o)), None)


@pytest.mark.parametrize("kw", [
    dict(n=-1), dict(rows=-1), dict(cap=-1), dict(pages=-1), dict(ld=3), dict(pages=1 << 27, ld=1 << 27),
    dict(t=None), dict(lengths=None), dict(counts=None), dict(free=None), dict(count=None),
    dict(words=1), dict(parents=P), dict(parents=P, words=1025), dict(parents=P, words=-1),
    dict(parents=P, words=1, out=dict(mask=None)), dict(out=dict(lengths=P + 256)),
    dict(out=dict(row_start=None)), dict(out=dict(requests=None)), dict(out=dict(positions=None)),
    dict(out=dict(slots=None)), dict(out=dict(lengths=None)), dict(out=dict(status=None)),
    dict(out=dict(free_count=None)), dict(out=dict(page_start=None)),
])
def test_block_tables_refuses(kw):
    assert tables(**kw) == BAD
    assert b"block_tables" in _lib.lib().wl_last_error()


@pytest.mark.parametrize("kw", [
    dict(n=-1), dict(cap=-1), dict(pages=-1), dict(ld=3), dict(t=None), dict(lengths=None), dict(keep=None),
    dict(free=None), dict(count=None), dict(out=dict(lengths=None)), dict(out=dict(lengths=P + 256)),
    dict(out=dict(status=None)), dict(out=dict(free_count=None)), dict(out=dict(page_start=None)),
])
def test_release_pages_refuses(kw):
    a = dict(t=P, ld=4, pages=4, lengths=P, keep=P + 256, n=2, free=P, cap=4, count=P, out={})
    a.update(kw)
    o = dict(lengths=P + 512, status=P, free_count=P, page_start=P)
    o.update(a["out"])
    assert _lib.lib().wl_release_pages(a["t"], a["ld"], a["pages"], a["lengths"], a["keep"], a["n"], a["free"],
                                       a["cap"], a["count"], C.byref(_lib.ReleaseResult(**o)), None) == BAD


@pytest.mark.parametrize("kw,code", [
    (dict(rows=-1), BAD), (dict(hd=12), BAD), (dict(hd=0), BAD), (dict(kvh=0), BAD), (dict(pages=-1), BAD),
    (dict(pages=1 << 28), BAD), (dict(kvh=1 << 20), BAD), (dict(cache=0), UNS), (dict(cache=2), UNS),
    (dict(k=None), BAD), (dict(v=None), BAD), (dict(slots=None), BAD), (dict(ck=None), BAD), (dict(cv=None), BAD),
    (dict(k=ODD), BAD), (dict(v=ODD), BAD), (dict(ck=ODD), BAD), (dict(cv=ODD), BAD), (dict(ldk=127), BAD),
    (dict(ldv=64), BAD), (dict(ldk=130), BAD), (dict(src=1, ldk=132), BAD), (dict(src=30), UNS),
    (dict(src=2), UNS), (dict(src=1, cache=30), UNS), (dict(rows=0, k=None, v=None, slots=None), OK),
])
def test_kv_append_refuses(kw, code):
    a = dict(src=0, cache=1, k=P, v=P, ldk=128, ldv=128, slots=P, rows=1, kvh=2, hd=64, pages=1, ck=P, cv=P)
    a.update(kw)
    assert _lib.lib().wl_kv_append(*a.values(), None) == code


@pytest.mark.parametrize("kw,code", [
    (dict(n=-1), BAD), (dict(na=-1), BAD), (dict(hd=20), BAD), (dict(hd=1032), BAD), (dict(kvh=0), BAD),
    (dict(ld=1), BAD), (dict(pages=-1), BAD), (dict(cache=0), UNS), (dict(t=None), BAD), (dict(lengths=None), BAD),
    (dict(acc=None), BAD), (dict(start=None), BAD), (dict(ck=None), BAD), (dict(cv=None), BAD),
    (dict(ck=ODD), BAD), (dict(n=0, t=None), OK), (dict(na=0, acc=None), OK),
])
def test_kv_commit_refuses(kw, code):
    a = dict(cache=1, t=P, ld=2, max_pages=2, lengths=P, n=1, acc=P, start=P, na=1, kvh=2, hd=64, pages=1, ck=P,
             cv=P)
    a.update(kw)
    assert _lib.lib().wl_kv_commit(*a.values(), None) == code


@pytest.mark.parametrize("kw,code", [
    (dict(qt=2), UNS), (dict(qt=12), UNS), (dict(hd=96), UNS), (dict(hd=0), UNS), (dict(n=-1), BAD),
    (dict(rows=-1), BAD), (dict(heads=3), BAD), (dict(heads=0), BAD), (dict(kvh=0), BAD), (dict(ld=1), BAD),
    (dict(pages=-1), BAD), (dict(pages=1 << 27), BAD), (dict(window=-1), BAD), (dict(words=1), BAD),
    (dict(mask=P), BAD), (dict(mask=P, words=1025), BAD), (dict(scale=0.0), BAD), (dict(scale=-1.0), BAD),
    (dict(scale=float("nan")), BAD), (dict(scale=float("inf")), BAD), (dict(q=None), BAD), (dict(out=None), BAD),
    (dict(t=None), BAD), (dict(lengths=None), BAD), (dict(start=None), BAD), (dict(pos=None), BAD),
    (dict(ck=None), BAD), (dict(cv=None), BAD), (dict(ldq=255), BAD), (dict(ldq=257), BAD), (dict(q=ODD), BAD),
    (dict(out=ODD), BAD), (dict(ck=ODD), BAD), (dict(cv=ODD), BAD), (dict(ws=ODD), BAD),
    (dict(rows=0, q=None, out=None), OK), (dict(n=0, t=None), OK),
])
def test_tree_attention_refuses(kw, code):
    a = dict(qt=0, q=P, ldq=256, ck=P, cv=P, pages=1, t=P, ld=2, max_pages=2, lengths=P, start=P, pos=P, mask=None,
             words=0, n=1, rows=1, heads=4, kvh=2, hd=64, window=0, scale=0.125, out=P, ws=P, nb=1 << 40)
    a.update(kw)
    assert _lib.lib().wl_tree_attention(*a.values(), None) == code


def test_tree_attention_wants_its_workspace():
    need = _lib.lib().wl_tree_attention_workspace(0, 1, 1, 4, 2, 64)
    if need:
        args = [0, P, 256, P, P, 1, P, 2, 2, P, P, P, None, 0, 1, 1, 4, 2, 64, 0, 0.125, P]
        assert _lib.lib().wl_tree_attention(*args, P, need - 1, None) == SMALL
        assert _lib.lib().wl_tree_attention(*args, None, need, None) == SMALL
    assert _lib.lib().wl_tree_attention_workspace(0, 0, 1, 4, 2, 64) == 0
    assert _lib.lib().wl_tree_attention_workspace(0, 1, 1, 3, 2, 64) == 0


@pytest.mark.parametrize("kw,ctx,code", [
    (dict(type=2), {}, UNS), (dict(rows=-1), {}, BAD), (dict(V=0), {}, BAD), (dict(ld=9), {}, BAD),
    (dict(ldo=9), {}, BAD), (dict(logits=None), {}, BAD), (dict(out=None), {}, BAD), (dict(params=None), {}, BAD),
    (dict(out=P, ldo=11), {}, BAD), (dict(V=(1 << 27) + 1, ld=1 << 28, ldo=1 << 28), {}, BAD),
    ({}, dict(history=P), BAD), ({}, dict(prompt_lens=P), BAD), ({}, dict(history_start=P, history_total=3), BAD),
    ({}, dict(n_history=-1), BAD), ({}, dict(history_total=-1), BAD), ({}, dict(bias_total=-1), BAD),
    ({}, dict(n_allowed=-1), BAD), ({}, dict(draft_mask=P), BAD), ({}, dict(draft_tokens=P), BAD),
    ({}, dict(words=1), BAD), ({}, dict(draft_mask=P, draft_tokens=P, words=1), BAD),
    ({}, dict(draft_mask=P, draft_tokens=P, row_start=P, words=1025), BAD), ({}, dict(bias_tokens=P), BAD),
    ({}, dict(bias_start=P, bias_total=2), BAD), ({}, dict(allowed=P, n_allowed=1, allowed_words=0), BAD),
    (dict(rows=0, logits=None, out=None, params=None), {}, OK),
])
def test_process_logits_refuses(kw, ctx, code):
    a = dict(type=0, logits=P, ld=10, rows=1, V=10, params=P, out=P + 1024, ldo=10)
    a.update(kw)
    c = _lib.LogitContext(**ctx)
    assert _lib.lib().wl_process_logits(a["type"], a["logits"], a["ld"], a["rows"], a["V"], a["params"],
                                        C.byref(c), a["out"], a["ldo"], None) == code


def test_python_checks():
    t = torch.zeros(2, 4, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        ops.block_tables(t, t[0], t[0], t[0], t[0], 4)
    with pytest.raises(ValueError, match="CUDA"):
        ops.kv_append(t, t, t, t, t)
    with pytest.raises(ValueError, match="CUDA"):
        ops.tree_attention(t, t, t, t, t, t, t)
    with pytest.raises(ValueError, match="CUDA"):
        ops.process_logits(t.float(), t)
    for kw in (dict(repetition=0.0), dict(repetition=[1.0, -2.0]), dict(repetition=float("inf")),
               dict(presence=float("nan")), dict(frequency=float("inf"))):
        with pytest.raises(ValueError):
            ops.logit_params(2, device="cpu", **kw)
    rec = ops.logit_params(3, [1.0, 2.0, 3.0], 0.5, allowed_row=[-1, 0, 7], device="cpu").numpy().view("<f4")
    assert rec.reshape(3, 4)[:, 0].tolist() == [1, 2, 3] and rec.view("<i4").reshape(3, 4)[:, 3].tolist() == [-1, 0, 7]
