"""roundtrip of host data: numpy out, in the type that came in."""
import numpy as np
import pytest
import torch

from oracle import mx_oracle as O

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [np.float16, np.float32, np.float64])
def test_roundtrip_keeps_the_type(dtype):
    from perm_amd import mxfp4
    x = np.random.default_rng(1).standard_normal((3, 5, 64)).astype(dtype)
    want = O.mx_values(*O.mx_quantize(x.astype(np.float32).reshape(15, 64))).reshape(x.shape).astype(dtype)
    for given in (x, torch.from_numpy(x)):
        y = mxfp4.roundtrip(given)
        assert isinstance(y, np.ndarray) and y.dtype == dtype and np.array_equal(y, want)


def test_roundtrip_of_other_types_is_float32():
    from perm_amd import mxfp4
    x = torch.arange(64).reshape(2, 32)
    for given in (x, x.numpy(), x.tolist(), x.to(torch.bfloat16)):
        y = mxfp4.roundtrip(given)
        assert y.dtype == np.float32 and y.shape == (2, 32)
