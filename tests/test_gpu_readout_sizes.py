"""GPU tests of the read-out loss at sizes where its kernels change: rows of the network's 2,333 columns and of up to 2^16, lists of up to
1,024 columns, one position, and a network's loss of odd batches.  Against the float64 oracle within its bounds."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from test_gpu_readout import DEV, TYPES, call, case, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,d,v", [(100, 1025, 65), (101, 2333, 70), (97, 2560, 33), (130, 3101, 66), (97, 4099, 40), (98, 1 << 16, 3),
                                      (1, 2333, 4168), (33, 4096, 50), (5, 1 << 16, 130), (64, 2333, 200)])
def test_long_rows(rows, d, v, dtype):
    t = case(rows, d, v, dtype, seed=d, k=2, legal=True)
    check(call(*t, grad_scale=0.25), t, dtype, np.full(rows, 0.25))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows", [3, 100, 300])
@pytest.mark.parametrize("k", [33, 64, 65, 1000, 1024])
def test_long_lists(rows, k, dtype):
    """More targets than a wave has lanes, columns repeated among them."""
    t = case(rows, 40, 700, dtype, seed=k, k=k, legal=True, index=torch.int32)
    check(call(*t), t, dtype)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows", [2, 98])
def test_many_columns(rows, dtype):
    """Lists at the first and the last of 2^20 columns, most of which no row sees: the gradients of those are 0."""
    v, d = 1 << 20, 3
    g = torch.Generator().manual_seed(rows)
    x, some = torch.randn(rows, d, generator=g).to(TYPES[dtype]), torch.tensor([0, 1, 31, 32, 4097, v // 2, v - 33, v - 2, v - 1])
    w = torch.randn(v, d, generator=g).to(TYPES[dtype])
    index = torch.randint(0, len(some), (rows, 2), generator=g)
    weight = torch.rand(rows, 2, generator=g)
    legal = torch.zeros(rows, v, dtype=torch.bool)
    legal[:, some] = True
    loss, grads = call(x, w, None, some[index], weight, legal)
    check((loss, grads._replace(weight=grads.weight[some.to(DEV)])), (x, w[some], None, index, weight, None), dtype)
    rest = torch.ones(v, dtype=torch.bool, device=DEV)
    rest[some.to(DEV)] = False
    assert not grads.weight[rest].any()


@pytest.mark.parametrize("batch", [1, 2, 97])
def test_a_networks_loss_of_odd_batches(batch):
    """One position and half-precision boards; moves as int32, rows' losses; the sum is theirs."""
    from chessfly.encoding import N_MOVES
    from chessfly.synthetic import GraphSpec, synthetic_boards, synthetic_net
    net, _ = synthetic_net(GraphSpec(n=1500, edges=40_000, n_sensory=150, n_output=60, seed=5), steps=3, seed=0, device=DEV)
    net.eval()
    x = torch.as_tensor(synthetic_boards(batch, seed=1), dtype=torch.float16, device=DEV)
    target = torch.randint(0, N_MOVES, (batch,), generator=torch.Generator().manual_seed(1)).to(torch.int32).to(DEV)
    sides = []
    for what in ("loss", "logits"):
        net.zero_grad(set_to_none=True)
        if what == "loss":
            rows, wdl = net.policy_loss(x, target, reduction="none")
            total, _ = net.policy_loss(x, target, reduction="sum")
            assert torch.equal(total, rows.sum())
        else:
            logits, wdl = net(x)
            rows = torch.nn.functional.cross_entropy(logits, target.long(), reduction="none")
        (rows.sum() + wdl.sum()).backward()
        sides.append((rows.detach(), wdl.detach(), {n: p.grad for n, p in net.named_parameters()}))
    (a, wa, ga), (b, wb, gb) = sides
    # as for a training batch: float32 sums of some 200 terms on both sides
    assert torch.equal(wa, wb) and ((a - b).abs() <= 2.0 ** -18 * b.abs()).all()
    for n in gb:
        assert (ga[n] - gb[n]).norm() <= 2.0 ** -13 * gb[n].norm(), n
