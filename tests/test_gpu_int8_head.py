"""GPU tests of the network's 8-bit read-out and of the distillation example that runs the operators together."""

from __future__ import annotations

import importlib.util
import os

import numpy as np
import pytest
import torch

from helpers import PKG

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _net(dtype, steps=4):
    from chessfly.synthetic import GraphSpec, synthetic_net
    net, _ = synthetic_net(GraphSpec(n=3000, edges=120_000, n_sensory=300, n_output=100, seed=8), steps=steps, seed=0,
                           device=DEV)
    net.eval()
    net.infer_dtype = dtype
    with torch.no_grad():
        net.norm.mean.normal_(0, 0.2)
        net.norm.var.uniform_(0.5, 2.0)
        net.policy_from.weight.normal_(0, 0.1)
        net.policy_to.weight.normal_(0, 0.1)
    return net


def _bound(net, weight, r):
    """|sum r w - sum q s p t| for operands each off by at most half a step, s / 2 and t / 2."""
    s, t = r.abs().amax(1) / 127, weight.abs().amax(1) / 127
    k = r.shape[1]
    return (t / 2) * r.abs().sum(1)[:, None] + (s / 2)[:, None] * weight.abs().sum(1) + k * s[:, None] * t / 4


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("batch", [1, 37])
def test_int8_head_is_within_half_a_step_of_the_float_head(dtype, batch):
    from chessfly.synthetic import synthetic_boards
    net = _net(dtype)
    x = torch.as_tensor(synthetic_boards(batch, seed=3), device=DEV)
    with torch.no_grad():
        logits, wdl = net(x)
        net.head_dtype = torch.int8
        logits8, wdl8 = net(x)
        net.infer_dtype = torch.float32
        u = (torch.nn.functional.linear(x[:, :838].float(), net.encoder.weight[:, :838], net.encoder.bias) * 5.0).T.contiguous()
        r = net.norm(net.brain.forward_io(u, net.in_idx, net.out_idx, net.cfg.steps).T).double()
        w = (net.policy.weight + net.policy_from.weight[net.move_from] + net.policy_to.weight[net.move_to]).double()
    # the float head is itself within 1e-3 of the float32 path (both state dtypes), and so is the half drive
    assert logits8.shape == logits.shape and logits8.is_contiguous() and wdl8.is_contiguous()
    assert bool(((logits8 - logits).abs().double() <= _bound(net, w, r) * 1.001 + 2e-3).all())
    assert bool(((wdl8 - wdl).abs().double() <= _bound(net, net.value.weight.double(), r) * 1.001 + 2e-3).all())
    assert float((logits8 - logits).abs().max()) > 0          # it is another path


def test_int8_head_follows_the_weights_and_serves_the_evaluator():
    from chessfly.model import Evaluator
    from chessfly.synthetic import synthetic_boards
    net = _net(torch.float16)
    net.head_dtype = torch.int8
    x = synthetic_boards(12, seed=3)
    evaluate = Evaluator(net, torch.device(DEV))
    policy, values = evaluate(x.astype(np.float16), None, None)
    with torch.no_grad():
        logits, wdl = net(torch.as_tensor(x, device=DEV))
        assert np.array_equal(policy, logits.half().cpu().numpy())
        assert np.allclose(values, net.expected_value(wdl).cpu().numpy(), atol=1e-6)
        before = logits.clone()
        net.policy.bias.add_(1.0)
        after, _ = net(torch.as_tensor(x, device=DEV))
        assert torch.allclose(after, before + 1.0, atol=1e-4)
        assert net(torch.as_tensor(x[:0], device=DEV))[0].shape == (0, 4168)
        net.head_dtype = torch.bfloat16
        with pytest.raises(RuntimeError, match="head_dtype"):
            net(torch.as_tensor(x, device=DEV))


def test_training_ignores_the_head_dtype():
    from chessfly.synthetic import synthetic_boards
    net = _net(torch.float32)
    net.train()
    x = torch.as_tensor(synthetic_boards(4, seed=3), device=DEV)
    ref = net(x)[0].detach()
    net.norm.mean.zero_()
    net.head_dtype = torch.int8
    out = net(x)[0]
    assert out.requires_grad and ref.shape == out.shape


def test_label_wants_a_teacher_in_eval_mode():
    from chessfly.distill import label
    net = _net(torch.float16)
    net.train()
    with pytest.raises(RuntimeError, match="eval"):
        label(net, torch.zeros(2, 838, device=DEV), 4)


def test_example_student_learns():
    path = os.path.join(PKG, "examples", "distill.py")
    spec = importlib.util.spec_from_file_location("distill_example", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    losses = example.run(steps=24, batch=64, say=lambda *_: None)
    assert all(np.isfinite(losses)) and min(losses) >= 0
    assert np.mean(losses[-4:]) < 0.5 * np.mean(losses[:4])
