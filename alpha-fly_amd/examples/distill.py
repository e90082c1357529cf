"""A student network learns from a teacher's labels.

The teacher evaluates positions with its read-out in 8 bits and keeps each position's best legal moves and the log-sum-exp of
the rest (chessfly.distill.label); the student, with fewer recurrent steps, trains on those lists and on the teacher's
win/draw/loss probabilities.  Synthetic graph and boards:

    python alpha-fly_amd/examples/distill.py --steps 40 --batch 256
"""

from __future__ import annotations

import argparse
import os
import sys

import numpy as np
import torch
import torch.nn.functional as F

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))

from chessfly.distill import distill_loss, label  # noqa: E402
from chessfly.encoding import N_MOVES  # noqa: E402
from chessfly.synthetic import GraphSpec, synthetic_boards, synthetic_net  # noqa: E402


def legal_moves(batch: int, seed: int, device) -> torch.Tensor:
    """About 30 legal moves a position."""
    legal = np.random.default_rng([seed, 0x1E6A]).random((batch, N_MOVES)) < 30 / N_MOVES
    legal[:, 0] = True
    return torch.as_tensor(legal, device=device)


def run(steps: int = 40, batch: int = 256, moves: int = 24, temperature: float = 2.0, spec: GraphSpec | None = None,
        device: str = "cuda:0", say=print) -> list[float]:
    """The policy losses of the steps, one training batch each."""
    spec = spec or GraphSpec(n=4000, edges=200_000, n_sensory=400, n_output=120, seed=7)
    teacher, conn = synthetic_net(spec, steps=6, seed=0, device=device)
    teacher.eval()
    teacher.head_dtype = torch.int8
    student, _ = synthetic_net(spec, steps=4, seed=1, device=device, graph=conn)
    student.train()
    optimiser = torch.optim.AdamW(student.parameters(), lr=3e-3, weight_decay=0.0)
    losses = []
    for step in range(steps):
        x = torch.as_tensor(synthetic_boards(batch, seed=step % 4), dtype=torch.float32, device=device)
        legal = legal_moves(batch, step % 4, device)
        lists, wdl = label(teacher, x, moves, temperature, legal)        # a replay buffer would keep these
        logits, student_wdl = student(x)
        policy = distill_loss(logits, lists, temperature, legal)
        value = F.cross_entropy(student_wdl, wdl.softmax(-1))
        optimiser.zero_grad(set_to_none=True)
        (policy + value).backward()
        torch.nn.utils.clip_grad_norm_(student.parameters(), 5.0)
        optimiser.step()
        losses.append(policy.detach())
    losses = [float(v) for v in torch.stack(losses)]
    say(f"policy divergence {losses[0]:.4f} -> {losses[-1]:.4f} over {steps} steps of {batch} positions")
    return losses


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    parser.add_argument("--steps", type=int, default=40)
    parser.add_argument("--batch", type=int, default=256)
    parser.add_argument("--moves", type=int, default=24, help="moves that the teacher's lists keep (1 to 256)")
    parser.add_argument("--temperature", type=float, default=2.0)
    a = parser.parse_args()
    run(a.steps, a.batch, a.moves, a.temperature)
