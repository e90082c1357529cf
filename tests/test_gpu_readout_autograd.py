"""GPU tests of the read-out loss under autograd: what it has no gradient for, and which graphs of its leaves a capture finds."""

from __future__ import annotations

import pytest
import torch

from test_gpu_readout import DEV, FEW, MANY, case, on

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [FEW, MANY])
def test_the_targets_weights_have_no_gradient(rows):
    """Weights that are learnt too: the loss and the other gradients are the same, a backward pass to the weights raises."""
    from chessfly.readout import Visits, readout_loss
    x, w, b, index, weight, legal = on(*case(rows, 33, 70, "float32", k=3, legal=True))
    w.requires_grad_()
    plain = readout_loss(x, w, b, Visits(index, weight), legal)
    (want,) = torch.autograd.grad(plain, w)
    learnt = weight.clone().requires_grad_()
    for share in (learnt, learnt.softmax(1).mul(0).add(weight)):      # a leaf, and what is computed from one
        loss = readout_loss(x, w, b, Visits(index, share), legal)
        assert torch.equal(loss, plain)
        assert torch.equal(torch.autograd.grad(loss, w, retain_graph=True)[0], want)
        with pytest.raises(RuntimeError, match="targets' weights has no backward"):
            loss.backward()
        alone = readout_loss(x, w.detach(), b, Visits(index, share), legal)
        assert torch.equal(alone, plain)
        with pytest.raises(RuntimeError, match="targets' weights has no backward"):
            alone.backward()
    assert learnt.grad is None
    assert torch.equal(readout_loss(x, w.detach(), b, Visits(index, learnt.detach()), legal), plain)
    with torch.no_grad():
        assert not readout_loss(x, w, b, Visits(index, learnt), legal).requires_grad


def test_the_targets_weights_have_no_forward_derivative():
    from torch.autograd import forward_ad
    from chessfly.readout import Visits, readout_loss
    x, w, b, index, weight, _ = on(*case(20, 9, 12, "float32", k=3))
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        readout_loss(x, w, b, Visits(index, forward_ad.make_dual(weight, torch.ones_like(weight))))
