"""The loss operators at the edges of their arguments: empty and expanded
inputs, forward-mode derivatives, temperatures below 1, values near the types'
limits, upstream gradients of rows that count for nothing.

Definitions and tolerances are those of ``test_gpu_losses``; where a test has a
bound of its own, the reason stands beside it.
"""

import math

import pytest
import torch

from pytorch_opt_b200 import _lib, losses
from tests.test_gpu_losses import DTYPES, GRAD_TOL, _gen, _grads, _head, _loss_bound, _rel, _teacher, ref_ce, ref_distill

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _no_device_error(cuda):
    yield
    assert _lib.device_error(reset=True) == 0


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("top,temperature", [(1, 1.0), (3, 1.0), (1, 2.0), (5, 0.5)])
def test_linear_distillation_empty(top, temperature, reduction):
    w = torch.randn(10, 8, device="cuda").requires_grad_()
    h = torch.empty(0, 8, device="cuda").requires_grad_()
    i, t = torch.empty(0, top, dtype=torch.long, device="cuda"), torch.empty(0, top, device="cuda")
    loss = losses.linear_distillation(h, w, i, t, temperature=temperature, reduction=reduction)
    gh, gw = _grads(loss, h, w, up=torch.ones_like(loss))
    assert gh.shape == (0, 8) and (gw == 0).all()
    if reduction == "none":
        assert loss.shape == (0,)
    else:
        assert float(loss.detach()) == 0.0


def test_forward_mode_is_refused():
    """No tangent is lost silently: a dual tensor without requires_grad is refused like any other."""
    h, w, y = _head(20, 64, 300, torch.float32, seed=1)
    index, teacher = _teacher(20, 300, 3, 2)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(h, torch.ones_like(h))
        for reduction in ("mean", "none"):
            for call in (lambda a: losses.linear_cross_entropy(a, w, y, reduction=reduction),
                         lambda a: losses.linear_cross_entropy(h, torch.autograd.forward_ad.make_dual(w, w), y),
                         lambda a: losses.linear_distillation(a, w, index, teacher, reduction=reduction),
                         lambda a: losses.distillation(a, index.clamp(max=63), teacher, reduction=reduction)):
                with pytest.raises(RuntimeError):  # (NotImplementedError is one)
                    call(dual)
                with torch.no_grad(), pytest.raises(RuntimeError):  # which does not stop forward mode
                    call(dual)
        plain = losses.linear_cross_entropy(h, w, y)  # no dual among its inputs
    assert torch.equal(plain, losses.linear_cross_entropy(h, w, y))
