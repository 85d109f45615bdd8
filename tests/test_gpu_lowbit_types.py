"""Arguments that are missing or of a wrong kind, refused with the modules' own errors."""
import numpy as np
import pytest
import torch

from test_gpu_kvcache import _i32, kv  # noqa: F401

pytestmark = pytest.mark.gpu


def test_lengths_are_needed(kv):  # noqa: F811
    c = kv.new(4, 2, 64, 16)
    k = torch.zeros((2, 2, 64), dtype=torch.bfloat16, device="cuda")
    t, n = _i32([[0], [1]]), _i32([0, 0])
    with pytest.raises(ValueError, match="filled"):
        kv.write(c, k, k, t, None)
    with pytest.raises(ValueError, match="lens"):
        kv.attention(k, c, t, None)
    with pytest.raises(ValueError, match="table"):
        kv.attention(k, c, None, n)
    with pytest.raises(TypeError):
        kv.attention(k, c, t, n, window=1.5)


def test_rows_are_tensors(kv):  # noqa: F811
    from perm_amd import mxfp4
    c = kv.new(4, 2, 64, 16)
    x = np.zeros((2, 2, 64), np.float32)
    k = torch.zeros((2, 2, 64), dtype=torch.bfloat16, device="cuda")
    t, n = _i32([[0], [1]]), _i32([0, 0])
    for bad in (x, x.tolist(), None):
        with pytest.raises(TypeError):
            kv.write(c, bad, bad, t, n)
        with pytest.raises(TypeError):
            kv.write(c, k, bad, t, n)
        with pytest.raises(TypeError):
            kv.attention(bad, c, t, n)
        with pytest.raises(TypeError):
            mxfp4.linear(bad, mxfp4.quantize(k[0]))
    with pytest.raises(TypeError):
        mxfp4.dequantize(k)
    with pytest.raises(TypeError):
        mxfp4.matmul(mxfp4.quantize(k[0]), k)
    with pytest.raises(TypeError):
        kv.read((c.k, c.v), t, _i32([0, 1, 2]), 2)
