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


@pytest.mark.parametrize("temperature", [0.0, -1.0, float("nan"), float("inf"), 1e-39, 2.0**-61, 2.0**61])
def test_abi_refuses_temperatures_outside_fp32(temperature):
    lib = _lib.load()
    assert lib.po_linear_loss(P, 8, P, 8, 0, 4, 8, 16, P, 2, P, 2, 0, 2, -100, 0.0, 0.0, temperature, 1, None, P, P,
                              None, 8, None, 8, 0, P, 1 << 30, None) == 1
    assert "temperature" in _lib.last_error()
    assert lib.po_distill_logits(P, 16, 0, 4, 16, P, 2, P, 2, 0, 2, temperature, 1, None, P, P, None, 16, P, 8,
                                 None) == 1
    assert "temperature" in _lib.last_error()


def test_abi_refuses_row_grad_beside_a_scaled_scalar():
    lib = _lib.load()
    for mode in (2, 3):
        assert lib.po_distill_logits(P, 16, 1, 4, 16, P, 2, P, 2, 0, 2, 1.0, mode, P, P, P, P, 16, P, 8, None) == 1
        assert "row_grad" in _lib.last_error()
        assert lib.po_linear_loss(P, 8, P, 8, 2, 4, 8, 16, P, 1, None, 1, 0, 1, -100, 0.0, 0.0, 1.0, mode, P, P, P, P, 8,
                                  None, 8, 0, P, 1 << 30, None) == 1
        assert "row_grad" in _lib.last_error()
