"""GPU tests of the read-out loss and the clipping together: in a network's training step, in its example, in a captured step."""

from __future__ import annotations

import os
import runpy

import numpy as np
import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "alpha-fly_amd")


def _net(seed=0):
    from chessfly.synthetic import GraphSpec, synthetic_net
    net, _ = synthetic_net(GraphSpec(n=2000, edges=60_000, n_sensory=200, n_output=90, seed=3), steps=4, seed=seed, device=DEV)
    net.train()
    return net


def _batch(batch, seed=0):
    from chessfly.encoding import N_MOVES
    from chessfly.readout import Visits
    from chessfly.synthetic import synthetic_boards
    g = torch.Generator().manual_seed(seed)
    legal = torch.rand(batch, N_MOVES, generator=g) < 0.01
    index = torch.randint(0, N_MOVES, (batch, 12), generator=g)
    legal.scatter_(1, index, True)
    share = torch.rand(batch, 12, generator=g)
    share /= share.sum(1, keepdim=True)
    pi = torch.zeros(batch, N_MOVES).scatter_add_(1, index, share)
    x = torch.as_tensor(synthetic_boards(batch, seed=seed), dtype=torch.float32, device=DEV)
    result = torch.randint(0, 3, (batch,), generator=g)
    return x, Visits(index.to(torch.int32).to(DEV), share.to(DEV)), pi.to(DEV), legal.to(DEV), result.to(DEV)


@pytest.mark.parametrize("batch", [16, 200])
def test_a_networks_policy_loss_is_that_of_its_logits(batch):
    """The loss and every parameter's gradient, against torch's softmax over the network's own logits.  Both sides round to float32
    at every layer: a logit of up to 10 errs by some 200 sums of 2^-24 each, 2^-13 of the gradients in the norm at most."""
    x, visits, pi, legal, result = _batch(batch)
    sides = []
    for own in (True, False):
        net = _net()
        if own:
            policy, wdl = net.policy_loss(x, visits, legal)
        else:
            logits, wdl = net(x)
            policy = -(pi * logits.masked_fill(~legal, -1e9).log_softmax(-1)).sum(-1).mean()
        (policy + F.cross_entropy(wdl, result)).backward()
        sides.append((float(policy), wdl.detach(), {n: p.grad for n, p in net.named_parameters()}))
    (a, wa, ga), (b, wb, gb) = sides
    assert abs(a - b) <= 2.0 ** -18 * abs(b) and torch.equal(wa, wb)
    assert ga.keys() == gb.keys()
    for n in gb:
        assert (ga[n] - gb[n]).norm() <= 2.0 ** -13 * gb[n].norm(), n


def test_steps_with_clipping_follow_torchs():
    """Three steps of loss, backward, clipping and AdamW, each from the same weights: norms and clipped gradients."""
    from chessfly.clip import clip_grad_norm_
    net = _net(1)
    optimiser = torch.optim.AdamW(net.parameters(), lr=1e-3)
    for step in range(3):
        x, visits, _, legal, result = _batch(64, step)
        policy, wdl = net.policy_loss(x, visits, legal)
        optimiser.zero_grad(set_to_none=True)
        (policy + F.cross_entropy(wdl, result)).backward()
        grads = [p.grad.clone() for p in net.parameters()]
        limit = 0.5 * float(torch.cat([g.flatten() for g in grads]).double().norm())
        want = torch.cat([g.flatten() for g in grads]).double()
        norm = clip_grad_norm_(net.parameters(), limit)
        assert abs(float(norm) - want.norm()) <= 2.0 ** -23 * want.norm()
        got = torch.cat([p.grad.flatten() for p in net.parameters()]).double()
        assert ((got - 0.5 * want).abs() <= 1e-6 * want.abs() + 1e-38).all()
        optimiser.step()
    assert all(p.isfinite().all() for p in net.parameters())


def test_without_gradients_and_in_evaluation():
    """The loss of held-out positions: the layers in the network's inference type, the statistics left as they are."""
    net = _net().eval()
    x, visits, pi, legal, _ = _batch(33)
    net.infer_dtype = torch.float32
    with torch.no_grad():
        policy, wdl = net.policy_loss(x, visits, legal, reduction="none")
        logits, want = net(x)
    expected = -(pi * logits.masked_fill(~legal, -1e9).log_softmax(-1)).sum(-1)
    assert not policy.requires_grad and policy.shape == (33,)
    assert torch.allclose(policy, expected, rtol=1e-5, atol=1e-6) and torch.allclose(wdl, want, rtol=1e-4, atol=1e-5)
    with pytest.raises(RuntimeError, match="HIP device"):
        net.policy_loss(x.cpu(), visits, legal)


def test_a_networks_capture_beside_an_eager_graph_is_refused():
    """Before any layer runs: the layers' weights are leaves as well, and the read-out's own are none."""
    net = _net()
    x, visits, _, legal, _ = _batch(16)
    alive = net.policy_loss(x, visits, legal)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="still alive"):
        with torch.cuda.graph(graph):
            net.policy_loss(x, visits, legal)
    sum(t.sum() for t in alive).backward()
    assert all(p.grad.isfinite().all() for p in net.parameters())


@pytest.mark.parametrize("rows", [20, 300])
def test_a_captured_step(rows):
    """Loss, backward, clipping and an update in one graph, replayed between eager steps from the same weights."""
    from chessfly.clip import clip_grad_norm_
    from chessfly.readout import Visits, readout_loss
    g = torch.Generator().manual_seed(rows)
    lin = torch.nn.Linear(70, 150).to(DEV)
    x = torch.randn(rows, 70, generator=g).to(DEV)
    target = Visits(torch.randint(0, 150, (rows, 3), generator=g).to(DEV), torch.rand(rows, 3, generator=g).to(DEV))
    start = [p.detach().clone() for p in lin.parameters()]

    def step():
        loss = readout_loss(x, lin.weight, lin.bias, target)
        lin.weight.grad, lin.bias.grad = torch.autograd.grad(loss, (lin.weight, lin.bias))
        norm = clip_grad_norm_(lin.parameters(), 0.05)
        with torch.no_grad():
            for p in lin.parameters():
                p.sub_(p.grad)
        return loss.detach(), norm

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    captured = [p.grad for p in lin.parameters()]
    for seed in range(4):
        x.copy_(torch.randn(rows, 70, generator=torch.Generator().manual_seed(seed)))
        results = []
        for replay in (True, False):
            with torch.no_grad():
                for p, s in zip(lin.parameters(), start):
                    p.copy_(s)
            if replay:
                graph.replay()
                got = (*out, *captured)
            else:
                got = (*step(), *[p.grad for p in lin.parameters()])
            torch.cuda.synchronize()
            results.append([t.clone() for t in (*got, *lin.parameters())])
        assert all(torch.equal(a, b) for a, b in zip(*results))


def test_offsets_past_32_bits():
    """Rows over 2^31 elements apart, of few rows and of many."""
    from chessfly.readout import readout_loss_and_grad
    d, v = 40, 60
    for rows, apart in ((3, 1_150_000_000), (300, 8_000_000)):
        big = torch.empty((rows - 1) * apart + d, dtype=torch.bfloat16, device=DEV)
        far = big.as_strided((rows, d), (apart, 1))
        g = torch.Generator(device=DEV).manual_seed(1)
        x, w = torch.randn(rows, d, generator=g, device=DEV).bfloat16(), torch.randn(v, d, generator=g, device=DEV).bfloat16()
        t = torch.randint(0, v, (rows,), generator=g, device=DEV)
        far.copy_(x)
        a, b = readout_loss_and_grad(far, w, None, t), readout_loss_and_grad(x, w, None, t)
        assert torch.equal(a[0], b[0]) and all(torch.equal(p, q) for p, q in zip(a[1][:2], b[1][:2]))
        del big, far


def test_a_gradient_of_more_than_2_31_elements():
    from chessfly.clip import clip_grad_norm_
    n = (1 << 31) + 77
    p = torch.nn.Parameter(torch.empty(n, dtype=torch.float16, device=DEV))
    p.grad = torch.ones(n, dtype=torch.float16, device=DEV)
    p.grad[-1] = 100.0
    norm = clip_grad_norm_(p, 0.25 * float(np.sqrt(n - 1 + 1e4)))
    assert abs(float(norm) - np.sqrt(n - 1 + 1e4)) <= 2.0 ** -23 * float(norm)
    assert float(p.grad[-1]) == 25.0 and float(p.grad[n // 2]) == 0.25 and bool((p.grad[: 1 << 20] == 0.25).all())


def test_the_example_runs():
    run = runpy.run_path(os.path.join(PKG, "examples", "train.py"))["run"]
    said = []
    from chessfly.synthetic import GraphSpec
    seen = run(steps=3, batch=40, moves=8, limit=0.01, spec=GraphSpec(n=1500, edges=40_000, n_sensory=150, n_output=60, seed=5),
               say=said.append)
    assert len(seen) == 3 and len(said) == 1 and np.isfinite(seen).all() and all(norm > 0 for _, norm in seen)
