"""Operators without gradients: a backward pass to any input that wants one raises."""
import pytest
import torch

from perm_amd import _lib


@pytest.mark.parametrize("wants", [(True, False), (False, True), (True, True)])
def test_any_input_that_wants_a_gradient(wants):
    xs = [torch.ones(3).requires_grad_(w) for w in wants]
    y = _lib.no_backward(torch.ones(4), "an operator", *xs)
    assert y.requires_grad
    with pytest.raises(NotImplementedError, match="an operator"):
        y.sum().backward()
    with torch.no_grad():
        assert not _lib.no_backward(torch.ones(4), "an operator", *xs).requires_grad


def test_no_input_that_wants_a_gradient():
    y = torch.ones(4)
    assert _lib.no_backward(y, "an operator", torch.ones(3), None) is y
    assert _lib.no_backward(y, "an operator", torch.ones(3).requires_grad_(), None).requires_grad
