"""A network learns from a search's visits.

Each position comes with its legal moves, the visits that a search gave some of them, and the game's result; the policy's loss and
its gradients come from the read-out without keeping the logits (FlyChessNet.policy_loss), and the step is clipped by the norm of
all gradients.  Synthetic graph, boards and visits:

    python alpha-fly_amd/examples/train.py --steps 40 --batch 256
"""

from __future__ import annotations

import argparse
import os
import sys

import numpy as np
import torch
import torch.nn.functional as F

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))

from chessfly.clip import clip_grad_norm_  # noqa: E402
from chessfly.encoding import N_MOVES  # noqa: E402
from chessfly.readout import Visits  # noqa: E402
from chessfly.synthetic import GraphSpec, synthetic_boards, synthetic_net  # noqa: E402


def searched(batch: int, moves: int, seed: int, device):
    """Visits over up to `moves` of about 30 legal moves a position, the legal moves, and win, draw or loss."""
    rng = np.random.default_rng([seed, 0x5EA2C4])
    legal = rng.random((batch, N_MOVES)) < 30 / N_MOVES
    legal[:, 0] = True
    order = np.argsort(np.where(legal, rng.random(legal.shape), -1.0), axis=1)[:, ::-1][:, :moves]
    there = np.take_along_axis(legal, order, 1)
    share = np.where(there, rng.random(order.shape) ** 3, 0.0)
    share /= share.sum(1, keepdims=True)
    to = lambda a, t: torch.as_tensor(np.ascontiguousarray(a), dtype=t, device=device)
    visits = Visits(to(np.where(there, order, -1), torch.int32), to(share, torch.float32))
    return visits, to(legal, torch.bool), to(rng.integers(0, 3, batch), torch.int64)


def run(steps: int = 40, batch: int = 256, moves: int = 24, limit: float = 5.0, spec: GraphSpec | None = None,
        device: str = "cuda:0", say=print) -> list[tuple[float, float]]:
    """The policy loss and the gradients' norm of each step."""
    spec = spec or GraphSpec(n=4000, edges=200_000, n_sensory=400, n_output=120, seed=7)
    net, _ = synthetic_net(spec, steps=6, seed=0, device=device)
    net.train()
    optimiser = torch.optim.AdamW(net.parameters(), lr=3e-3, weight_decay=0.0)
    seen = []
    for step in range(steps):
        x = torch.as_tensor(synthetic_boards(batch, seed=step % 4), dtype=torch.float32, device=device)
        visits, legal, result = searched(batch, moves, step % 4, device)
        policy, wdl = net.policy_loss(x, visits, legal)
        optimiser.zero_grad(set_to_none=True)
        (policy + F.cross_entropy(wdl, result)).backward()
        norm = clip_grad_norm_(net.parameters(), limit)
        optimiser.step()
        seen.append((policy.detach(), norm))
    seen = [(float(a), float(b)) for a, b in seen]
    say(f"policy loss {seen[0][0]:.4f} -> {seen[-1][0]:.4f}, gradient norm {seen[0][1]:.3f} -> {seen[-1][1]:.3f} over {steps} steps of "
        f"{batch} positions")
    return seen


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    parser.add_argument("--steps", type=int, default=40)
    parser.add_argument("--batch", type=int, default=256)
    parser.add_argument("--moves", type=int, default=24, help="moves that the visits keep (1 to 1024)")
    parser.add_argument("--limit", type=float, default=5.0, help="the gradients' norm is clipped to this")
    a = parser.parse_args()
    run(a.steps, a.batch, a.moves, a.limit)
