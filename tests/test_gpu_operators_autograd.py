"""GPU tests of the operators without a derivative where autograd follows their inputs: the same results, and an error in place
of a gradient that is not there."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _calls():
    from chessfly.distill import top_logits
    from chessfly.int8 import Int8Linear, quantize_rows
    lin = Int8Linear.from_float(torch.randn(9, 12, device=DEV))
    q, s = quantize_rows(torch.randn(3, 12, device=DEV))
    x = torch.randn(3, 12, device=DEV)
    return {"quantize_rows": (lambda t: quantize_rows(t)[1], x), "Int8Linear": (lin, x),
            "Int8Linear scale": (lambda t: lin(q, scale=t), s),
            "top_logits": (lambda t: top_logits(t, 4).values, x), "top_logits tail": (lambda t: top_logits(t, 4).tail, x)}


@pytest.mark.parametrize("name", ["quantize_rows", "Int8Linear", "Int8Linear scale", "top_logits", "top_logits tail"])
def test_a_gradient_that_is_not_there_raises(name):
    call, x = _calls()[name]
    ref = call(x)
    assert not ref.requires_grad
    leaf = x.clone().requires_grad_(True)
    out = call(leaf)
    assert torch.equal(out, ref)
    with pytest.raises(RuntimeError, match="no backward pass"):
        (out.sum() + leaf.sum()).backward()
    with torch.no_grad():
        assert torch.equal(call(leaf), ref) and not call(leaf).requires_grad
    with forward_ad.dual_level():
        assert torch.equal(call(x), ref)
        with pytest.raises(RuntimeError, match="forward-mode"):
            call(forward_ad.make_dual(x, torch.ones_like(x)))


def test_integer_results_and_labels_of_a_tracked_teacher():
    from chessfly.distill import TopLogits, distill_loss, top_logits
    from chessfly.int8 import quantize_rows
    t = torch.randn(3, 12, device=DEV, requires_grad=True)
    lists = top_logits(t, 4)
    assert type(lists) is TopLogits and not lists.index.requires_grad and lists.values.requires_grad
    assert top_logits(t, 4, tail=False).tail is None
    assert not quantize_rows(t)[0].requires_grad
    z = torch.randn(3, 12, device=DEV, requires_grad=True)
    distill_loss(z, lists).backward()            # the teacher is a constant of the loss
    assert z.grad is not None and t.grad is None


def test_the_loss_in_forward_mode_is_refused():
    from chessfly.distill import distill_loss, top_logits
    z = torch.randn(3, 12, device=DEV)
    lists = top_logits(torch.randn(3, 12, device=DEV), 4)
    with forward_ad.dual_level():
        assert torch.equal(distill_loss(z, lists), distill_loss(z, lists))
        with pytest.raises(RuntimeError):
            distill_loss(forward_ad.make_dual(z, torch.ones_like(z)), lists)


def test_the_loss_has_no_second_derivative():
    from chessfly.distill import distill_loss, top_logits
    z = torch.randn(3, 12, device=DEV, requires_grad=True)
    (grad,) = torch.autograd.grad(distill_loss(z, top_logits(torch.randn(3, 12, device=DEV), 4)), z, create_graph=True)
    with pytest.raises(RuntimeError):
        grad.sum().backward()
