"""Host-side checks of the loss operators at the edges of their arguments (no GPU)."""

import ctypes

import pytest
import torch

from pytorch_opt_b200 import _lib, losses

P = ctypes.c_void_p(256)  # never followed: every call below is refused or empty


@pytest.mark.parametrize("top,temperature", [(1, 1.0), (3, 1.0), (3, 2.0)])
def test_linear_loss_abi_takes_an_empty_call_of_either_kind(top, temperature):
    """No token, so no index, no hidden row, no teacher has an address, and nothing is left to launch."""
    status = _lib.load().po_linear_loss(None, 8, P, 8, 0, 0, 8, 16, None, top, None, top, 0, top, -100, 0.0, 0.0,
                                        temperature, 1, None, None, None, None, 8, None, 8, 0, None, 0, None)
    assert status == 0, _lib.last_error()


def test_dual_tensors_go_through_autograd():
    """Which refuses them; past it their tangent would be lost without a word."""
    x = torch.ones(2)
    assert not losses._records(x) and losses._records(x.clone().requires_grad_())
    with torch.autograd.forward_ad.dual_level(), torch.no_grad():
        assert losses._records(torch.autograd.forward_ad.make_dual(x, x))
    assert not losses._records(x)
