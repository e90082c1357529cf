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


def _net():
    from chessfly.synthetic import GraphSpec, synthetic_net
    net, _ = synthetic_net(GraphSpec(n=1500, edges=40_000, n_sensory=150, n_output=60, seed=5), steps=3, seed=0, device=DEV)
    return net.train()


def _mark(p):
    return torch.autograd.graph.get_gradient_edge(p).node.metadata.get("chessfly.stream")


@pytest.mark.parametrize("learns", ["all", "recurrence", "maps"])
@pytest.mark.parametrize("kept", ["logits", "wdl"])
def test_a_forwards_graph_is_found_by_a_capture(kept, learns):
    """An eager forward of the network whose results live: a captured policy_loss of the same leaves is refused before any layer
    runs.  Once they are dropped, nothing is left of it."""
    from chessfly.synthetic import synthetic_boards
    net = _net()
    for name, p in net.named_parameters():
        trunk = name.startswith(("encoder", "brain"))
        p.requires_grad_(learns == "all" or (name.startswith("brain") if learns == "recurrence" else not trunk))
    x = torch.as_tensor(synthetic_boards(8, seed=0), dtype=torch.float32, device=DEV)
    target = torch.zeros(8, dtype=torch.int64, device=DEV)
    marked = [p for p in net.parameters() if p.requires_grad]
    assert not any(_mark(p) is not None for p in marked)
    alive = net(x)[kept == "wdl"]
    assert any(_mark(p) is not None for p in marked)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="still alive"):
        with torch.cuda.graph(graph):
            net.policy_loss(x, target)
    alive.sum().backward()
    del alive
    assert not any(_mark(p) is not None for p in marked)
    with torch.no_grad():
        out = net(x)
    assert not any(_mark(p) is not None for p in marked) and out[0].isfinite().all()


def test_a_captured_forward_beside_an_eager_graph_still_runs():
    """Only its backward pass would wait for the other stream: the forward is marked, not refused."""
    from chessfly import _hip
    w = torch.ones(3, device=DEV, requires_grad=True)
    nodes = _hip.held_leaves("eager", w)
    torch.cuda.synchronize()
    graph, out = torch.cuda.CUDAGraph(), torch.zeros(3, device=DEV)
    with torch.cuda.graph(graph):
        assert _hip.held_leaves("captured", w, refuse=False)[0] is not None
        with pytest.raises(RuntimeError, match="captured: .* still alive"):
            _hip.held_leaves("captured", w)
        out.add_(w.detach())
    for n in range(1, 4):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, torch.full_like(out, float(n)))
    assert len(nodes) == 1 and _hip.held_leaves("host", torch.ones(2, requires_grad=True)) == []
