"""The operators for several answers at the edges of what their calls allow."""
import pytest
import torch

from test_gpu_kvcache import _i32, kv  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads", [4, 8])
def test_slopes_that_want_a_gradient(kv, heads):  # noqa: F811
    """Attention depends on its slopes: a backward pass to them alone raises, of results and log-sums."""
    c = kv.new(4, 2, 64, 16)
    t, n = _i32([[0], [1], [2]]), _i32([16] * 3)
    q = torch.ones((3, heads, 64), dtype=torch.bfloat16, device="cuda")
    slopes = torch.ones(heads, device="cuda").requires_grad_()
    plain = kv.attention(q, c, t, n, slopes=slopes.detach(), return_lse=True)
    for want, got in zip(plain, kv.attention(q, c, t, n, slopes=slopes, return_lse=True)):
        assert not want.requires_grad and got.requires_grad and torch.equal(want, got)
        with pytest.raises(NotImplementedError, match="attention"):
            got.float().sum().backward()
    with torch.no_grad():
        assert not kv.attention(q, c, t, n, slopes=slopes).requires_grad
