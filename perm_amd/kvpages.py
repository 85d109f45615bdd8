"""The pages of a cache (``perm_amd.kvcache``) as several answers to one prompt need them: shared,
handed out, given back and moved together, on the GPU.

The books are two int32 tensors, changed in place and never read by the host: table [batch,
max_pages], the page numbers of every sequence with -1 for no page, and refs [pages], how many
entries of the table hold each page. A page without holders is free. One pair of books serves
the caches of all layers of a model, whose pages have the same numbers.

  new(pages)                                     refs of a cache whose pages are all free
  fork(refs, table, lens, parents, children, block)   children share their parents' pages
  grow(refs, table, filled, new, block)          pages for the next tokens -> (src, dst, missing)
  copy(cache, src, dst)                          pages src[i] into pages dst[i], for every layer
  free(refs, table, rows)                        sequences' pages given back
  compact(refs, table)                           pages in use to the front -> (src, dst, used)

A step of several answers: ``free`` those that ended, ``fork`` a prompt's row into others, then
before each ``kvcache.write`` call ``grow`` and, for each layer's cache, ``copy``: a page that
sequences share and one of them is about to write into becomes its own.

The books of a call are its own until it is done: one stream at a time. What a call does is
fixed by its inputs, whatever the order in which the GPU's workgroups run.
"""
import ctypes
import operator

import torch

from . import _lib
from .kvcache import BLOCKS, _desc


def new(pages, device="cuda"):
    """refs [pages] of a cache whose pages are all free (a table of them is all -1)."""
    if pages < 1:
        raise ValueError(f"{pages} pages")
    return torch.zeros((pages,), dtype=torch.int32, device=device)


def _ints(t, dims, what, device, size=None):
    """An int32 CUDA tensor of ``dims`` dimensions (of ``size``, where it has one)."""
    if not (isinstance(t, torch.Tensor) and t.is_cuda):
        raise ValueError(f"{what} must be a CUDA tensor")
    if t.device != device:
        raise ValueError(f"{what} is on {t.device}, not {device}")
    if t.dtype != torch.int32 or t.dim() != dims:
        raise IndexError(f"{what} must be int32 with {dims} dimension(s), got {t.dtype} "
                         f"{tuple(t.shape)}")
    if size is not None and t.shape[0] != size:
        raise ValueError(f"{what} of {t.shape[0]}, not {size}")
    return t if t.is_contiguous() else t.contiguous()


def _books(refs, table):
    """The two checked: they are changed in place, so neither is copied."""
    for t, dims, what in ((refs, 1, "refs"), (table, 2, "table")):
        if _ints(t, dims, what, getattr(refs, "device", None)) is not t:
            raise ValueError(f"{what} is changed in place and must be contiguous")
    _lib.here(refs)
    return refs.data_ptr(), refs.shape[0], table.data_ptr(), table.shape[0], table.shape[1]


def _block(block):
    if block not in BLOCKS:
        raise ValueError(f"pages of {block} tokens: one of {BLOCKS}")
    return int(block)


def fork(refs, table, lens, parents, children, block):
    """Row children[i] of the table becomes row parents[i] as far as its lens[parents[i]] tokens
    go, and -1 past them; the pages gain a holder each. parents and children: int32 [n]. A child's row
    should hold no pages (``free`` it first), is named once and is no parent of the same call.
    Numbers that are no row of the table are left out, and a row into itself. lens (int32 [batch]) is read alone: the
    children's lengths are the caller's to set."""
    lib = _lib.load()
    books = _books(refs, table)
    lens = _ints(lens, 1, "lens", refs.device, table.shape[0])
    children = _ints(children, 1, "children", refs.device)
    parents = _ints(parents, 1, "parents", refs.device, children.shape[0])
    _lib.check(lib.cp_kv_fork(*books, lens.data_ptr(), _block(block), parents.data_ptr(),
                              children.data_ptr(), children.shape[0], _lib.stream_ptr()))


def grow(refs, table, filled, new, block):
    """Pages for the next new[b] tokens of sequence b, which holds filled[b] (int32 [batch]; new
    may be a number for all): (src, dst, missing), int32 [batch] each.

    An entry that those tokens fall into gets a page where it has none, and one of its own where
    other sequences hold its page too. Holders count as before the call: where all of a page's are
    to write into it, each gets a page, and theirs is free after the call. Only the first entry
    can hold tokens already: src[b] and dst[b] then name the pages that ``copy`` has to copy, and
    are -1 otherwise; such an entry without a page stays as it is. Free pages are handed out by
    number, to the sequences in order, until one wants more than there are: it and the ones after
    it that want any get none, and missing[b] says how many they wanted (also for tokens past the
    table's end). Write no rows of such a sequence: its last page may be another's too."""
    lib = _lib.load()
    books = _books(refs, table)
    batch = table.shape[0]
    filled = _ints(filled, 1, "filled", refs.device, batch)
    each = 0
    if isinstance(new, torch.Tensor):
        new = _ints(new, 1, "new", refs.device, batch)
    else:
        each, new = operator.index(new), None
        if not 0 <= each < 2 ** 31:
            raise ValueError(f"{each} tokens")
    src, dst, missing = (refs.new_empty((batch,)) for _ in range(3))
    nws = lib.cp_kv_grow_ws_bytes(refs.shape[0], batch)
    ws = _lib.workspace(nws, refs.device)
    _lib.check(lib.cp_kv_grow(*books, filled.data_ptr(), _lib.ptr(new), each, _block(block),
                              src.data_ptr(), dst.data_ptr(), missing.data_ptr(), _lib.ptr(ws),
                              nws, _lib.stream_ptr()))
    return src, dst, missing


def free(refs, table, rows=None):
    """The pages of these rows of the table (int32 [n]; None: of all) lose a holder, the rows
    become -1. Numbers that are no row are left out; a row named twice counts once."""
    lib = _lib.load()
    books = _books(refs, table)
    if rows is not None:
        rows = _ints(rows, 1, "rows", refs.device)
        if rows.shape[0] == 0:
            return
    _lib.check(lib.cp_kv_free(*books, _lib.ptr(rows), 0 if rows is None else rows.shape[0],
                              _lib.stream_ptr()))


def compact(refs, table):
    """The pages in use numbered 0 to used - 1: those past that, in order, take the free numbers
    before it, in order. refs and table follow; (src, dst, used) with src and dst int32
    [pages // 2] for ``copy``, -1 past the last pair, and used int32 [1]. Every table that
    holds pages of refs has to be the one given."""
    lib = _lib.load()
    books = _books(refs, table)
    src, dst = (refs.new_empty((refs.shape[0] // 2,)) for _ in range(2))
    used = refs.new_empty((1,))
    nws = lib.cp_kv_compact_ws_bytes(refs.shape[0])
    ws = _lib.workspace(nws, refs.device)
    _lib.check(lib.cp_kv_compact(*books, src.data_ptr(), dst.data_ptr(), used.data_ptr(),
                                 _lib.ptr(ws), nws, _lib.stream_ptr()))
    return src, dst, used


def copy(cache, src, dst, into=None):
    """Codes and scales of page src[i] of the cache to page dst[i] of it, or of ``into``, a cache
    of the same heads, head dimension and block. Pairs with a number that is no page are left
    out. No page may be written twice in a call, nor one that it reads."""
    lib = _lib.load()
    desc = _desc(cache)
    to = desc if into is None else _desc(into)
    device = cache[0].device
    at = _lib.here(*cache, *(into or ()))
    src = _ints(src, 1, "src", device)
    dst = _ints(dst, 1, "dst", device, src.shape[0])
    _lib.check(lib.cp_kv_copy(ctypes.byref(desc), ctypes.byref(to), src.data_ptr(), dst.data_ptr(),
                              src.shape[0], _lib.stream_ptr(at)))
