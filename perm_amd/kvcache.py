"""A paged key / value cache in 8 bits, and attention over it, on the GPU.

Keys and values are held as e4m3 codes with one power-of-two scale for each page (a block of
tokens) and head. A sequence's position p is slot p % block of page table[b][p // block].

  new(pages, heads, head_dim, block)             an empty KvCache
  write(cache, k, v, table, filled, offsets)     quantizes and appends rows
  read(cache, table, offsets, total, dtype)      the tokens held, back in floating point
  attention(q, cache, table, lens, offsets)      softmax(q K^T) V over the codes

Ragged batches: ``offsets`` int32 [batch + 1] gives each sequence's first row of k, v or q;
None means one row a sequence, as in decoding. table int32 [batch, max_pages], filled and
lens int32 [batch] stay on the GPU and are read there: a call never waits for the device. An
entry of table outside the cache's pages is no page: what is written there is dropped, it
reads as 0, and attention does not see its tokens. Offsets do not decrease; rows before the
first and past the last (a padded batch) have no sequence: write leaves them out, read and
attention give 0 there.

For inference: rows written keep no graph, and a backward pass through attention raises
NotImplementedError.
"""
import ctypes
import operator
from typing import NamedTuple

import torch

from . import _lib
from .mxfp4 import DTYPES

BLOCKS = (16, 32, 64, 128)


class KvCache(NamedTuple):
    """k uint8 [pages, heads, block, head_dim], v uint8 [pages, heads, head_dim, block] (e4m3
    codes, V by column), k_scale and v_scale float32 [pages, heads]: powers of two between
    2^-60 and 2^60, the least that holds the page's largest value in +-448 codes."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor


def new(pages, heads, head_dim, block=16, device="cuda"):
    """An empty cache: code 0 and scale 1 everywhere."""
    if block not in BLOCKS or head_dim % 16 or not 16 <= head_dim <= 256 or min(pages, heads) < 1:
        raise ValueError(f"no cache of {pages} pages, {heads} heads of {head_dim}, {block} tokens "
                         f"a page: head_dim a multiple of 16 up to 256, block one of {BLOCKS}")
    u8 = dict(dtype=torch.uint8, device=device)
    return KvCache(torch.zeros((pages, heads, block, head_dim), **u8),
                   torch.zeros((pages, heads, head_dim, block), **u8),
                   torch.ones((pages, heads), device=device),
                   torch.ones((pages, heads), device=device))


def _desc(c):
    """struct cp_kv_cache of a KvCache, its buffers checked against each other."""
    if not (isinstance(c, (tuple, list)) and len(c) == 4):
        raise TypeError(f"cache must be a KvCache, got {type(c).__name__}")
    k, v, ks, vs = c
    if k.dim() != 4:
        raise ValueError("k codes are [pages, heads, block, head_dim]")
    pages, heads, block, d = k.shape
    if v.shape != (pages, heads, d, block) or ks.shape != (pages, heads) \
            or vs.shape != (pages, heads):
        raise ValueError(f"cache buffers of {tuple(k.shape)}, {tuple(v.shape)}, "
                         f"{tuple(ks.shape)}, {tuple(vs.shape)} do not fit")
    if k.dtype != torch.uint8 or v.dtype != torch.uint8 \
            or ks.dtype != torch.float32 or vs.dtype != torch.float32:
        raise TypeError("cache codes are uint8 and scales float32")
    if not (k.is_cuda and v.is_cuda and ks.is_cuda and vs.is_cuda and k.is_contiguous()
            and v.is_contiguous() and ks.is_contiguous() and vs.is_contiguous()):
        raise ValueError("cache buffers must be contiguous and on the GPU")
    return _lib.KvCacheDesc(k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), pages,
                            heads, block, d)


def _index(t, dims, what):
    """An int32 CUDA tensor of ``dims`` dimensions, contiguous."""
    if not (isinstance(t, torch.Tensor) and t.is_cuda):
        raise ValueError(f"{what} must be a CUDA tensor")
    if t.dtype != torch.int32 or t.dim() != dims:
        raise IndexError(f"{what} must be int32 with {dims} dimension(s), got {t.dtype} "
                         f"{tuple(t.shape)}")
    return t if t.is_contiguous() else t.contiguous()


def _batch(table, per_seq, what, offsets, rows):
    """table, per_seq and offsets as the kernels read them, their shapes checked."""
    table = _index(table, 2, "table")
    if what:
        per_seq = _index(per_seq, 1, what)
        if per_seq.shape[0] != table.shape[0]:
            raise ValueError(f"{what} of {per_seq.shape[0]} for {table.shape[0]} sequences")
    if offsets is not None:
        offsets = _index(offsets, 1, "offsets")
        if offsets.shape[0] != table.shape[0] + 1:
            raise ValueError(f"{offsets.shape[0]} offsets for {table.shape[0]} sequences")
    elif rows != table.shape[0]:
        raise ValueError(f"{rows} rows for {table.shape[0]} sequences need offsets")
    return table, per_seq, offsets


def _dtype(x, what):
    """The element type of a tensor."""
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{what} must be a tensor, got {type(x).__name__}")
    return x.dtype


def _heads(x, heads, d, what):
    """x [rows, heads, d] in strides the kernels read in place (copied where they cannot)."""
    if not x.is_cuda:
        raise ValueError(f"{what} must be on the GPU")
    if x.dim() != 3 or x.shape[2] != d or (heads is not None and x.shape[1] != heads):
        raise ValueError(f"{what} is {tuple(x.shape)}: [rows, {heads or 'heads'}, {d}]")
    step = 16 // x.element_size()
    if x.stride(2) != 1 or x.stride(0) % step or x.stride(1) % step or x.data_ptr() % 16:
        x = x.clone(memory_format=torch.contiguous_format)
    return x


def write(cache, k, v, table, filled, offsets=None):
    """Appends the rows of k and v [rows, heads, head_dim] (float32, bfloat16 or float16) to
    the cache in place: sequence b's rows go to positions filled[b], filled[b] + 1, ... A page
    begun in the call gets the scale of its own rows; one that holds tokens keeps its scale
    or moves to a larger one, its codes with it. Infinities saturate and, like NaN (kept as
    NaN), do not enter a scale. Sequences of one call must not share a page they write."""
    lib = _lib.load()
    desc = _desc(cache)
    dtype = _dtype(k, "k")
    if dtype != _dtype(v, "v") or dtype not in DTYPES:
        raise TypeError(f"k and v must both be float32, bfloat16 or float16, got {dtype}, "
                        f"{v.dtype}")
    k = _heads(k, desc.heads, desc.head_dim, "k")
    v = _heads(v, desc.heads, desc.head_dim, "v")
    rows = k.shape[0]
    if v.shape[0] != rows:
        raise ValueError(f"{rows} keys and {v.shape[0]} values")
    table, filled, offsets = _batch(table, filled, "filled", offsets, rows)
    if table.shape[0] == 0:
        return
    _lib.check(lib.cp_kv_write(
        ctypes.byref(desc), k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0),
        v.stride(1), DTYPES[dtype], rows, table.data_ptr(), table.shape[0], table.shape[1],
        filled.data_ptr(), _lib.ptr(offsets), _lib.stream_ptr()))


def read(cache, table, offsets, total, dtype=torch.bfloat16):
    """(k, v) [total, heads, head_dim] of ``dtype``: the first offsets[b + 1] - offsets[b]
    tokens of every sequence, at rows offsets[b] onward; total = offsets[-1], known to the
    caller."""
    lib = _lib.load()
    desc = _desc(cache)
    if dtype not in DTYPES:
        raise TypeError(f"dtype must be float32, bfloat16 or float16, got {dtype}")
    if offsets is None:
        raise ValueError("read needs offsets")
    table, _, offsets = _batch(table, None, "", offsets, total)
    shape = total, desc.heads, desc.head_dim
    k = cache.k.new_empty(shape, dtype=dtype)
    v = torch.empty_like(k)
    _lib.check(lib.cp_kv_read(ctypes.byref(desc), table.data_ptr(), table.shape[0],
                              table.shape[1], offsets.data_ptr(), total, k.data_ptr(),
                              v.data_ptr(), DTYPES[dtype], _lib.stream_ptr()))
    return k, v


def attention(q, cache, table, lens, offsets=None, *, causal=True, window=0, scale=None,
              return_lse=False):
    """softmax(scale * q K^T) V over the cache: q [rows, q heads, head_dim] in bfloat16 or
    float16 -> the same shape and type (and, with return_lse, float32 [rows, q heads]: the
    natural log of each row's sum of exponentials).

    Sequence b holds lens[b] tokens, and its query rows are its last ones (write them first):
    row i of n sits at position lens[b] - n + i and sees the tokens up to its own (causal) and,
    with window > 0, no more than the window's last ones. Query head x reads cache head
    x // (q heads / cache heads). scale is positive, head_dim ** -0.5 by default. A row that sees
    nothing, or has no sequence, is 0, its lse -inf."""
    lib = _lib.load()
    desc = _desc(cache)
    if _dtype(q, "q") not in (torch.bfloat16, torch.float16):
        raise TypeError(f"q must be bfloat16 or float16, got {q.dtype}")
    q = _heads(q, None, desc.head_dim, "q")
    rows, heads = q.shape[0], q.shape[1]
    if heads == 0 or heads % desc.heads:
        raise ValueError(f"{heads} query heads over {desc.heads} cache heads")
    window = min(operator.index(window), 2 ** 31 - 1)  # positions are below
    if window < 0:
        raise ValueError(f"window {window}")
    table, lens, offsets = _batch(table, lens, "lens", offsets, rows)
    out = torch.empty_like(q) if q.is_contiguous() else q.new_empty(q.shape)
    lse = torch.empty((rows, heads), device=q.device) if return_lse else None
    batch, max_pages = table.shape
    ragged = offsets is not None
    nws = lib.cp_kv_attention_ws_bytes(ctypes.byref(desc), rows, heads, batch, max_pages, ragged,
                                       window)
    ws = _lib.workspace(nws, q.device) if nws else None
    _lib.check(lib.cp_kv_attention(
        ctypes.byref(desc), q.data_ptr(), q.stride(0), q.stride(1), DTYPES[q.dtype], rows, heads,
        table.data_ptr(), batch, max_pages, lens.data_ptr(), _lib.ptr(offsets), int(causal),
        window, desc.head_dim ** -0.5 if scale is None else float(scale), out.data_ptr(),
        _lib.ptr(lse), _lib.ptr(ws), nws, _lib.stream_ptr()))
    out = _lib.no_backward(out, "kvcache.attention", q)
    return (out, _lib.no_backward(lse, "kvcache.attention", q)) if return_lse else out
