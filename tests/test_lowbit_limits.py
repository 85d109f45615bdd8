"""Sizes at which the cache's kernels would leave 32 bits: refused before anything is launched."""
import ctypes

import pytest

from perm_amd import _lib
from test_lowbit_args import P, _cache, lib  # noqa: F401


def _attend(lib, cache, rows, batch, max_pages, heads=4, window=0):
    return lib.cp_kv_attention(ctypes.byref(cache), P, 256, 64, 1, rows, heads, P, batch, max_pages, P, P, 1, window,
                               1.0, P, None, None, 0, None)


@pytest.mark.parametrize("block", [16, 32, 64, 128])
def test_tokens_of_a_sequence(lib, block):  # noqa: F811
    """Attention looks up pages of up to 240 tokens past a sequence's end in 32 bits."""
    most = 2 ** 31 // block
    for pages, status in ((most, _lib.CP_ERR_SHAPE), (most - 1, _lib.CP_ERR_SHAPE),
                          ((2 ** 31 - 1024) // block, _lib.CP_ERR_WORKSPACE)):
        if pages <= 2 ** 24 - 1:  # tables are no wider
            assert _attend(lib, _cache(block=block), 300, 1, pages) == status, pages
            assert _attend(lib, _cache(block=block), 1, 1, pages) == status, pages


def test_rows(lib):  # noqa: F811
    c = ctypes.byref(_cache(heads=1))
    for rows in (2 ** 31 - 1, 2 ** 31 - 200):
        assert lib.cp_kv_read(c, P, 1, 2, P, rows, P, P, 1, None) == _lib.CP_ERR_SHAPE
        assert lib.cp_kv_write(c, P, 64, 64, P, 64, 64, 1, rows, P, 1, 2, P, P, None) == _lib.CP_ERR_SHAPE
        assert _attend(lib, _cache(heads=1), rows, 1, 2, heads=1) == _lib.CP_ERR_SHAPE


def test_work_items_of_a_launch(lib):  # noqa: F811
    """A launch holds under 2^32 work items, 2^24 workgroups of 256."""
    c = ctypes.byref(_cache(heads=64))
    rows = 2 ** 24 + 64  # a wave a head and 16 rows or a page of 16
    assert lib.cp_kv_read(c, P, 1, 2, P, rows, P, P, 1, None) == _lib.CP_ERR_SHAPE
    assert lib.cp_kv_write(c, P, 64, 64, P, 64, 64, 1, rows, P, 1, 2, P, P, None) == _lib.CP_ERR_SHAPE
    # tiles of 16 rows: a workgroup a sequence and head
    assert _attend(lib, _cache(heads=64), 2 ** 18 + 64, 2 ** 18 + 64, 1, heads=64) == _lib.CP_ERR_SHAPE
    # the product: 16 columns of up to 16 waves, and tiles of up to eight waves
    for m, n in ((1, 2 ** 27), (2 ** 21, 2 ** 21)):
        assert lib.cp_mx4_matmul(P, P, m, P, P, n, 32, P, 1, P, 1 << 50, None) == _lib.CP_ERR_SHAPE
