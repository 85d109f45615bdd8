"""The low-bit entry points' argument checks, which answer before the device is touched."""
import ctypes

import pytest

from perm_amd import _lib

P = 1 << 20  # a non-null, aligned address that no refused call reads


@pytest.fixture(scope="module")
def lib():
    return _lib.load(require_gpu=False)


def _cache(**kw):
    f = dict(k=P, v=P, k_scale=P, v_scale=P, pages=4, heads=2, block=16, head_dim=64)
    f.update(kw)
    return _lib.KvCacheDesc(*(f[n] for n, _ in _lib.KvCacheDesc._fields_))


def _quantize(lib, x=P, dt=1, rows=4, k=64, stride=64, codes=P, scales=P):
    return lib.cp_mx4_quantize(x, dt, rows, k, stride, codes, scales, None)


@pytest.mark.parametrize("kw,status", [
    (dict(k=48), _lib.CP_ERR_SHAPE), (dict(k=0), _lib.CP_ERR_SHAPE), (dict(rows=-1), _lib.CP_ERR_SHAPE),
    (dict(stride=32), _lib.CP_ERR_SHAPE), (dict(dt=3), _lib.CP_ERR_ARG), (dict(x=None), _lib.CP_ERR_ARG),
    (dict(codes=None), _lib.CP_ERR_ARG), (dict(x=P + 8), _lib.CP_ERR_ALIGN),
    (dict(stride=68), _lib.CP_ERR_ALIGN), (dict(codes=P + 4), _lib.CP_ERR_ALIGN),
    (dict(scales=P + 2), _lib.CP_ERR_ALIGN), (dict(rows=0, x=None, codes=None, scales=None), _lib.CP_OK)])
def test_quantize(lib, kw, status):
    assert _quantize(lib, **kw) == status
    assert status == _lib.CP_OK or lib.cp_last_error()


@pytest.mark.parametrize("kw,status", [
    (dict(n=-1), _lib.CP_ERR_SHAPE), (dict(k=33), _lib.CP_ERR_SHAPE), (dict(ydt=5), _lib.CP_ERR_ARG),
    (dict(y=None), _lib.CP_ERR_ARG), (dict(y=P + 4), _lib.CP_ERR_ALIGN), (dict(nws=16), _lib.CP_ERR_WORKSPACE),
    (dict(ws=None), _lib.CP_ERR_WORKSPACE), (dict(ws=P + 16), _lib.CP_ERR_ALIGN), (dict(m=0), _lib.CP_OK),
    (dict(n=0), _lib.CP_OK)])
def test_linear(lib, kw, status):
    a = dict(m=40, n=8, k=64, ydt=1, y=P, ws=P, nws=1 << 20)
    a.update(kw)
    got = lib.cp_mx4_linear(P, 1, a["m"], 64, P, P, a["n"], a["k"], a["y"], a["ydt"], a["ws"], a["nws"], None)
    assert got == status


def test_few_rows_need_no_workspace(lib):
    assert lib.cp_mx4_linear_ws_bytes(4, 8, 64) == 0 and lib.cp_mx4_linear_ws_bytes(33, 8, 64) > 0
    assert lib.cp_mx4_linear_ws_bytes(4, 8, 1 << 20) > 0
    assert lib.cp_mx4_matmul_ws_bytes(100, 4096, 14336) > 0 == lib.cp_mx4_matmul_ws_bytes(16, 4096, 14336)


def _write(lib, cache, rows=3, batch=3, dt=1, k=P, k_row=128, k_head=64, offsets=None, table=P,
           max_pages=2, filled=P):
    return lib.cp_kv_write(ctypes.byref(cache), k, k_row, k_head, P, 128, 64, dt, rows, table, batch,
                           max_pages, filled, offsets, None)


@pytest.mark.parametrize("kw,status", [
    (dict(block=48), _lib.CP_ERR_SHAPE), (dict(block=8), _lib.CP_ERR_SHAPE), (dict(head_dim=72), _lib.CP_ERR_SHAPE),
    (dict(head_dim=272), _lib.CP_ERR_SHAPE), (dict(heads=0), _lib.CP_ERR_SHAPE), (dict(pages=0), _lib.CP_ERR_SHAPE),
    (dict(k=None), _lib.CP_ERR_ARG), (dict(v=P + 1), _lib.CP_ERR_ALIGN)])
def test_cache_descriptor(lib, kw, status):
    assert _write(lib, _cache(**kw)) == status
    assert lib.cp_kv_read(ctypes.byref(_cache(**kw)), P, 1, 2, P, 8, P, P, 1, None) == status
    assert lib.cp_kv_attention(ctypes.byref(_cache(**kw)), P, 256, 64, 1, 1, 4, P, 1, 2, P, None, 1, 0,
                               1.0, P, None, P, 1 << 30, None) == status


@pytest.mark.parametrize("kw,status", [
    (dict(rows=4), _lib.CP_ERR_SHAPE), (dict(max_pages=0), _lib.CP_ERR_SHAPE), (dict(batch=-1), _lib.CP_ERR_SHAPE),
    (dict(table=None), _lib.CP_ERR_ARG), (dict(filled=None), _lib.CP_ERR_ARG), (dict(k=None), _lib.CP_ERR_ARG),
    (dict(dt=7), _lib.CP_ERR_ARG), (dict(k_row=132), _lib.CP_ERR_ALIGN), (dict(k=P + 2), _lib.CP_ERR_ALIGN),
    (dict(k_head=-64), _lib.CP_ERR_SHAPE), (dict(rows=0, batch=0, table=None), _lib.CP_OK)])
def test_write(lib, kw, status):
    assert _write(lib, _cache(), **kw) == status


@pytest.mark.parametrize("kw,status", [
    (dict(heads=3), _lib.CP_ERR_SHAPE), (dict(heads=0), _lib.CP_ERR_SHAPE), (dict(dt=0), _lib.CP_ERR_ARG),
    (dict(window=-1), _lib.CP_ERR_ARG), (dict(lens=None), _lib.CP_ERR_ARG), (dict(q=P + 8), _lib.CP_ERR_ALIGN),
    (dict(rows=2), _lib.CP_ERR_SHAPE), (dict(max_pages=4096, nws=64), _lib.CP_ERR_WORKSPACE),
    (dict(rows=0, batch=0), _lib.CP_OK)])
def test_attention(lib, kw, status):
    a = dict(q=P, dt=1, rows=1, heads=4, batch=1, max_pages=2, lens=P, window=0, nws=1 << 30)
    a.update(kw)
    got = lib.cp_kv_attention(ctypes.byref(_cache()), a["q"], 256, 64, a["dt"], a["rows"], a["heads"], P,
                              a["batch"], a["max_pages"], a["lens"], None, 1, a["window"], 1.0, P, None, P,
                              a["nws"], None)
    assert got == status


def test_layout_sizes(lib):
    from perm_amd import mxfp4
    for rows, k in ((1, 32), (64, 128), (65, 160), (14336, 4096)):
        s = mxfp4.scale_shape(rows, k)
        n = 1
        for d in s:
            n *= d
        assert lib.cp_mx4_scale_bytes(rows, k) == n
