"""The next token of every row of a model's logits, on the GPU.

  sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0)   -> int32 [rows]

Random numbers are the caller's: u holds one of [0, 1) for each row, and the same logits, settings
and numbers give the same tokens, in whatever batch the row stands.

A token of logit x weighs e^((x - max) / temperature). Tokens are ordered by falling logit, equal
ones by rising number, and kept are

  top_k   the first k of them (0: all),
  top_p   of those, the ones before which less than top_p of their summed weight lies,
  min_p   of those, the ones that weigh at least min_p times the first;

the first always. In the order of their numbers, the token is the first one at which the sum of
the kept weights passes u times the whole of it. temperature 0 takes the first in the order. A NaN
counts as minus infinity, which is never chosen; a row that holds nothing else gives -1.

Weights are whole multiples of 2^-44 of the largest (151936 tokens; of up to 2^-51 in smaller
vocabularies) and their sums exact, so no token hangs on the order of additions.
"""
import operator

import torch

from . import _lib
from .mxfp4 import DTYPES


def _setting(v, rows, dtype, what, low, high, device):
    """(tensor or None, number): a setting of each row, or one for all."""
    if isinstance(v, torch.Tensor):
        if v.device != device:
            raise ValueError(f"{what} must be a number or on {device}")
        if v.dtype != dtype or v.shape != (rows,):
            raise ValueError(f"{what} of each row must be {dtype} [{rows}], got {v.dtype} "
                             f"{tuple(v.shape)}")
        return v.contiguous(), 0
    v = operator.index(v) if dtype == torch.int32 else float(v)
    if not low <= v <= high:
        raise ValueError(f"{what} {v} is not in [{low}, {high}]")
    return None, v


def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Tokens int32 [rows] of logits [rows, vocab] (float32, bfloat16 or float16; rows may be
    strided) and u [rows] (float32 or float64, in [0, 1)). A setting is a number, or a tensor
    [rows] (float32; top_k int32), whose entries out of range count as the nearest in it."""
    lib = _lib.load()
    code = DTYPES.get(logits.dtype) if isinstance(logits, torch.Tensor) else None
    if code is None:
        raise TypeError(f"logits must be float32, bfloat16 or float16, got "
                        f"{getattr(logits, 'dtype', type(logits).__name__)}")
    if not logits.is_cuda:
        raise ValueError("logits must be on the GPU")
    if logits.dim() != 2 or logits.shape[1] < 1:
        raise ValueError(f"logits are [rows, vocab], got {tuple(logits.shape)}")
    dev = logits.device
    at = _lib.here(logits)
    rows, vocab = logits.shape
    if not isinstance(u, torch.Tensor) or u.device != dev or u.shape != (rows,):
        raise ValueError(f"u must be a tensor [{rows}] on {dev}")
    if u.dtype not in (torch.float32, torch.float64):
        raise TypeError(f"u must be float32 or float64, got {u.dtype}")
    t, t_all = _setting(temperature, rows, torch.float32, "temperature", 0.0, float("inf"), dev)
    k, k_all = _setting(top_k, rows, torch.int32, "top_k", 0, 2 ** 31 - 1, dev)
    p, p_all = _setting(top_p, rows, torch.float32, "top_p", 0.0, 1.0, dev)
    m, m_all = _setting(min_p, rows, torch.float32, "min_p", 0.0, 1.0, dev)
    if logits.stride(1) != 1 and vocab > 1:
        logits = logits.contiguous()
    u = u.contiguous()
    token = logits.new_empty((rows,), dtype=torch.int32)
    nws = lib.cp_sample_ws_bytes(rows, vocab)
    ws = _lib.workspace(nws, dev)
    _lib.check(lib.cp_sample(logits.data_ptr(), code, rows, vocab, logits.stride(0), u.data_ptr(),
                             int(u.dtype == torch.float64), _lib.ptr(t), t_all, _lib.ptr(k), k_all,
                             _lib.ptr(p), p_all, _lib.ptr(m), m_all, token.data_ptr(),
                             _lib.ptr(ws), nws, _lib.stream_ptr(at)))
    return token
