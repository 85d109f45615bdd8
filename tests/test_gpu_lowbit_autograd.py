"""The low-bit operators have no gradients: a backward pass through them says so, and the
results are otherwise those without a graph."""
import pytest
import torch

from test_gpu_kvcache import _i32, kv  # noqa: F401

pytestmark = pytest.mark.gpu


def _check(call, x):
    with torch.no_grad():
        want = call(x)
    assert not want.requires_grad and not call(x.detach()).requires_grad
    y = call(x)
    assert y.requires_grad and torch.equal(y, want)
    with pytest.raises(NotImplementedError, match="backward"):
        y.float().sum().backward()
    y = call(x)
    y += 1  # in place, as on any result
    with pytest.raises(NotImplementedError):
        (2 * y).float().sum().backward()
    assert x.grad is None


@pytest.mark.parametrize("m", [1, 40])
def test_products(m):
    from perm_amd import mxfp4
    w = mxfp4.quantize(torch.nn.Parameter(torch.randn((48, 64), device="cuda")))
    x = torch.randn((m, 64), device="cuda", dtype=torch.bfloat16).requires_grad_()
    _check(lambda t: mxfp4.linear(t, w), x)
    _check(mxfp4.roundtrip, x)
    assert not mxfp4.dequantize(mxfp4.quantize(x)).requires_grad


def test_attention(kv):  # noqa: F811
    c = kv.new(4, 2, 64, 16)
    k = torch.randn((5, 2, 64), device="cuda", dtype=torch.bfloat16).requires_grad_()
    kv.write(c, k, k, _i32([[1]]), _i32([0]), _i32([0, 5]))
    q = torch.randn((5, 4, 64), device="cuda", dtype=torch.bfloat16).requires_grad_()
    args = (c, _i32([[1]]), _i32([5]), _i32([0, 5]))
    _check(lambda t: kv.attention(t, *args), q)
    _check(lambda t: kv.attention(t, *args, return_lse=True)[1], q)
