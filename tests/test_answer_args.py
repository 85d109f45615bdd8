"""Argument checks of the page and sampling entry points, which answer before the device is touched."""
import ctypes

import pytest

from perm_amd import _lib
from test_lowbit_args import P, _cache, lib  # noqa: F401

OK, SHAPE, ARG, ALIGN, WS = (_lib.CP_OK, _lib.CP_ERR_SHAPE, _lib.CP_ERR_ARG, _lib.CP_ERR_ALIGN,
                             _lib.CP_ERR_WORKSPACE)

BOOKS = [(dict(pages=0), SHAPE), (dict(pages=2 ** 31), SHAPE), (dict(max_pages=0), SHAPE), (dict(batch=-1), SHAPE),
         (dict(max_pages=2 ** 24), SHAPE), (dict(refs=None), ARG), (dict(table=None), ARG), (dict(refs=P + 2), ALIGN),
         (dict(table=P + 1), ALIGN)]


def _books(kw):
    a = dict(refs=P, pages=64, table=P, batch=3, max_pages=4)
    a.update({k: v for k, v in kw.items() if k in a})
    return a["refs"], a["pages"], a["table"], a["batch"], a["max_pages"]


@pytest.mark.parametrize("kw,status", BOOKS + [
    (dict(block=24), SHAPE), (dict(n=-1), SHAPE), (dict(n=2 ** 31), SHAPE), (dict(n=2 ** 24), SHAPE), (dict(lens=None), ARG),
    (dict(parents=None), ARG), (dict(children=None), ARG), (dict(n=0, lens=None), OK), (dict(batch=0, table=None), OK)])
def test_fork(lib, kw, status):  # noqa: F811
    a = dict(lens=P, block=16, parents=P, children=P, n=2)
    a.update(kw)
    assert lib.cp_kv_fork(*_books(kw), a["lens"], a["block"], a["parents"], a["children"], a["n"], None) == status
    assert status == OK or lib.cp_last_error()


@pytest.mark.parametrize("kw,status", BOOKS + [
    (dict(n=-1), SHAPE), (dict(n=2 ** 24), SHAPE), (dict(n=0), OK), (dict(batch=0, table=None), OK),
    (dict(rows=None, batch=0, table=None), OK), (dict(rows=None, batch=2 ** 24), SHAPE)])
def test_free(lib, kw, status):  # noqa: F811
    a = dict(rows=P, n=2)
    a.update(kw)
    assert lib.cp_kv_free(*_books(kw), a["rows"], a["n"], None) == status


@pytest.mark.parametrize("kw,status", BOOKS + [
    (dict(block=0), SHAPE), (dict(filled=None), ARG), (dict(src=None), ARG), (dict(dst=None), ARG), (dict(missing=None), ARG),
    (dict(ws=None), WS), (dict(nws=64), WS), (dict(ws=P + 4), ALIGN), (dict(batch=0, table=None, ws=None), OK)])
def test_grow(lib, kw, status):  # noqa: F811
    a = dict(filled=P, fresh=P, block=16, src=P, dst=P, missing=P, ws=P, nws=1 << 30)
    a.update(kw)
    got = lib.cp_kv_grow(*_books(kw), a["filled"], a["fresh"], 1, a["block"], a["src"], a["dst"], a["missing"], a["ws"],
                         a["nws"], None)
    assert got == status


@pytest.mark.parametrize("kw,status", BOOKS + [
    (dict(src=None), ARG), (dict(dst=None), ARG), (dict(used=None), ARG), (dict(ws=None), WS), (dict(nws=64), WS),
    (dict(ws=P + 4), ALIGN)])
def test_compact(lib, kw, status):  # noqa: F811
    a = dict(src=P, dst=P, used=P, ws=P, nws=1 << 30)
    a.update(kw)
    assert lib.cp_kv_compact(*_books(kw), a["src"], a["dst"], a["used"], a["ws"], a["nws"], None) == status


def test_workspaces(lib):  # noqa: F811
    assert lib.cp_kv_grow_ws_bytes(0, 4) == lib.cp_kv_compact_ws_bytes(0) == 0
    for pages in (1, 1000, 300000):
        assert lib.cp_kv_grow_ws_bytes(pages, 7) >= 4 * (2 * pages + 2 * 7 + pages // 1024)
        assert lib.cp_kv_compact_ws_bytes(pages) >= 4 * (pages + pages // 1024)


@pytest.mark.parametrize("a,b,kw,status", [
    ({}, dict(heads=3), {}, SHAPE), ({}, dict(block=32), {}, SHAPE), ({}, dict(head_dim=80), {}, SHAPE),
    (dict(k=None), {}, {}, ARG), ({}, dict(v=P + 8), {}, ALIGN), ({}, {}, dict(n=-1), SHAPE), ({}, {}, dict(n=2 ** 23), SHAPE),
    ({}, {}, dict(src=None), ARG), ({}, {}, dict(dst=None), ARG), ({}, dict(pages=9), dict(n=0, src=None), OK)])
def test_copy(lib, a, b, kw, status):  # noqa: F811
    x = dict(src=P, dst=P, n=3)
    x.update(kw)
    got = lib.cp_kv_copy(ctypes.byref(_cache(**a)), ctypes.byref(_cache(**b)), x["src"], x["dst"], x["n"], None)
    assert got == status


@pytest.mark.parametrize("kw,status", [
    (dict(dt=3), ARG), (dict(vocab=0), SHAPE), (dict(vocab=2 ** 24 + 1), SHAPE), (dict(rows=-1), SHAPE),
    (dict(rows=2 ** 31), SHAPE), (dict(step=-1), SHAPE), (dict(logits=None), ARG), (dict(u=None), ARG), (dict(token=None), ARG),
    (dict(logits=P + 1), ALIGN), (dict(u=P + 4, u64=1), ALIGN), (dict(rows=0, logits=None), OK), (dict(ws=None), WS),
    (dict(nws=1024), WS), (dict(ws=P + 16), ALIGN)])
def test_sample(lib, kw, status):  # noqa: F811
    a = dict(logits=P, dt=1, rows=2, vocab=100, step=100, u=P, u64=0, token=P, ws=P, nws=1 << 30)
    a.update(kw)
    got = lib.cp_sample(a["logits"], a["dt"], a["rows"], a["vocab"], a["step"], a["u"], a["u64"], None, 1.0, None, 0, None,
                        1.0, None, 0.0, a["token"], a["ws"], a["nws"], None)
    assert got == status


@pytest.mark.parametrize("kw,status", [
    (dict(heads=3), SHAPE), (dict(dt=0), ARG), (dict(window=-1), ARG), (dict(lens=None), ARG), (dict(q=P + 8), ALIGN),
    (dict(rows=3), SHAPE), (dict(nws=64, shared=P), WS), (dict(ws=P + 8, shared=P), ALIGN), (dict(softcap=-1.0), ARG),
    (dict(softcap=float("nan")), ARG), (dict(softcap=float("inf")), ARG), (dict(softcap=1e-38), ARG), (dict(more=False), ARG),
    (dict(shared=P, groups=0), SHAPE), (dict(shared=P, groups=4), SHAPE), (dict(shared=P, groups=-1), SHAPE),
    (dict(rows=0, batch=0), OK), (dict(rows=2 ** 24, batch=2 ** 24, max_pages=1, shared=P, groups=1), SHAPE)])
def test_attention_more(lib, kw, status):  # noqa: F811
    a = dict(q=P, dt=1, rows=6, heads=4, batch=6, max_pages=2, lens=P, window=0, nws=1 << 50, ws=P, softcap=0.0, shared=None,
             groups=2, more=True)
    a.update(kw)
    m = _lib.KvMore(a["softcap"], None, None, None, a["shared"], a["groups"])
    got = lib.cp_kv_attention_more(ctypes.byref(_cache()), a["q"], 256, 64, a["dt"], a["rows"], a["heads"], P, a["batch"],
                                   a["max_pages"], a["lens"], None, 1, a["window"], 1.0, ctypes.byref(m) if a["more"] else None,
                                   P, None, a["ws"], a["nws"], None)
    assert got == status


def test_workspaces_of_common_pages(lib):  # noqa: F811
    c = ctypes.byref(_cache())
    plain = lib.cp_kv_attention_ws_bytes(c, 64, 4, 64, 512, 0, 0)
    assert lib.cp_kv_attention_more_ws_bytes(c, 64, 4, 64, 512, 0, 0, 0) == plain
    # two phases: two splits of every row and head at the least, and two counts
    assert lib.cp_kv_attention_more_ws_bytes(c, 64, 4, 64, 1, 0, 0, 1) >= 64 * 4 * (2 * (64 + 2) + 2) * 4
    assert lib.cp_kv_attention_more_ws_bytes(c, 0, 4, 64, 1, 0, 0, 1) == 0
    # many rows of many tokens: their row tiles in order, two numbers for each
    more = lib.cp_kv_attention_more_ws_bytes(c, 40000, 4, 2, 1024, 1, 0, 0)
    tiles = (40000 * 2) // 128 + 2 + 1
    assert more - lib.cp_kv_attention_ws_bytes(c, 40000, 4, 2, 1024, 1, 0) == 8 * tiles
