"""A training step's loss and clipping, as cases that can be timed and checked.

A policy read-out learns from visit counts: its logits over the legal moves, their softmax cross entropy and its gradients come
from the read-out's inputs and weights, and the logits are not kept.  The step's gradients are then clipped by their norm over
all parameters.

Kinds of work ("what"):
* loss  readout_loss (direction "loss": each row's loss) and readout_loss_and_grad (direction "gradient": the gradients of
        the inputs, the weight and the bias too), against one column a row ("index") or a list of columns with weights
        ("visits").
* clip  clip_grad_norm_: the norm of all parameters' gradients, and the gradients scaled in place where it passes the limit.
"""

from __future__ import annotations

import math
import os
import random
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "alpha-fly_amd"))

own = False

DEV = "cuda:0"
N_MOVES, N_OUT = 4168, 2333          # the policy's moves, the output neurons that it reads
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
LEGAL = 30                           # legal moves of a chess position, about

# The parameters of the whole network (166,700 neurons, 10.5 million synapses) and of the example's (4,000 neurons).
NETWORKS = {
    "whole": [(10_494_794,), (166_700,), (166_700,), (17_937, 967), (17_937,), (N_MOVES, N_OUT), (N_MOVES,), (3, N_OUT), (3,),
              (64, N_OUT), (64,), (64, N_OUT), (64,)],
    "example": [(197_000,), (4000,), (4000,), (400, 967), (400,), (N_MOVES, 120), (N_MOVES,), (3, 120), (3,), (64, 120), (64,),
                (64, 120), (64,)],
    # six layers of projections, gated feed-forward and gains, with an embedding: a language model's
    "layers": [(50_257, 1024)] + [s for _ in range(6) for s in
                                  [(2048, 2048)] * 4 + [(8192, 2048), (8192, 2048), (2048, 8192), (2048,), (2048,)]],
}


def _loss_case(name, rows, d, v, dtype, direction, targets, k=1, legal=False):
    return {"name": name, "what": "loss", "rows": rows, "d": d, "v": v, "dtype": dtype, "direction": direction,
            "targets": targets, "k": k, "legal": legal}


def _clip_case(name, network, dtype, clips, norm="2"):
    return {"name": name, "what": "clip", "network": network, "tensors": len(NETWORKS[network]), "total": 0, "sizes": 0,
            "dtype": dtype, "clips": clips, "norm": norm}


def listed():
    return [
        # one position of a game being replayed, judged by its visits
        _loss_case("one position", 1, N_OUT, N_MOVES, "f32", "loss", "visits", 32, True),
        # the last moves of a game, learnt from at once
        _loss_case("few positions", 13, N_OUT, N_MOVES, "f32", "gradient", "visits", 32, True),
        # the training loop's batch
        _loss_case("training batch", 256, N_OUT, N_MOVES, "f32", "gradient", "visits", 32, True),
        # held-out positions of the self-play batch's size
        _loss_case("held-out positions", 1120, N_OUT, N_MOVES, "f32", "loss", "visits", 24, True),
        # a batch of games in half precision against the moves that were played, an odd size
        _loss_case("half precision", 1003, N_OUT, N_MOVES, "f16", "gradient", "index"),
        # a large batch in the network's own precision
        _loss_case("large batch", 4096, N_OUT, N_MOVES, "f32", "gradient", "visits", 32, True),
        # the largest: a part of a replay buffer
        _loss_case("largest batch", 16384, N_OUT, N_MOVES, "bf16", "gradient", "visits", 32, True),
        # a vocabulary of words of odd size, some tokens left out
        _loss_case("vocabulary", 4096, 1024, 50257, "bf16", "gradient", "index"),
        # held-out tokens
        _loss_case("vocabulary, held out", 2051, 768, 32000, "f16", "loss", "index"),
        # the example's network: small tensors, where latency counts
        _clip_case("example's gradients", "example", "f32", True),
        # the whole network on an ordinary step, below the limit
        _clip_case("network's gradients", "whole", "f32", False),
        # a language model's gradients, above it
        _clip_case("layers' gradients", "layers", "bf16", True),
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    if rng.random() < 0.3:
        # up to 48 tensors of up to 400 million elements together
        return {"what": "clip", "network": "", "tensors": rng.randint(1, 48), "total": _log_uniform(rng, 1000, 400_000_000),
                "sizes": rng.randrange(1 << 30), "dtype": rng.choice(["f32", "f16", "bf16", "mixed"]),
                "clips": rng.random() < 0.5, "norm": rng.choice(["2", "2", "inf"])}
    d = rng.choice([N_OUT, _log_uniform(rng, 64, 4096)])
    v = rng.choice([N_MOVES, _log_uniform(rng, 300, 50257)])
    # no more work than the largest batch, no more logits than the vocabulary
    rows = _log_uniform(rng, 1, max(1, min(16384, 16384 * N_OUT * N_MOVES // (d * v), 4096 * 50257 // v)))
    targets = rng.choice(["index", "visits"])
    return {"what": "loss", "rows": rows, "d": d, "v": v, "dtype": rng.choice(list(DTYPES)),
            "direction": rng.choice(["loss", "gradient", "gradient"]), "targets": targets,
            "k": 1 if targets == "index" else _log_uniform(rng, 1, 64), "legal": v == N_MOVES and rng.random() < 0.5}


def _shapes(case):
    if case["network"]:
        return NETWORKS[case["network"]]
    # sizes spread over their logarithm, scaled to the total
    r = random.Random(case["sizes"])
    parts = [math.exp(r.uniform(0, 9)) for _ in range(case["tensors"])]
    return [(max(1, int(case["total"] * p / sum(parts))),) for p in parts]


def _types(case):
    r = random.Random(case["sizes"] + 1)
    return [DTYPES[case["dtype"] if case["dtype"] != "mixed" else r.choice(list(DTYPES))] for _ in _shapes(case)]


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed) & 0x7FFFFFFF)
    randn = lambda *s: torch.randn(*s, generator=gen, device=DEV)
    rand = lambda *s: torch.rand(*s, generator=gen, device=DEV)
    if case["what"] == "clip":
        # each parameter's gradient has a size of its own, from 1e-4 to 1e-2; the limit is half or twice the norm, about
        params = [torch.nn.Parameter(torch.empty(s, dtype=t, device=DEV)) for s, t in zip(_shapes(case), _types(case))]
        r = random.Random(case["sizes"] + 2)
        scales = [10.0 ** r.uniform(-4, -2) for _ in params]
        for p, s in zip(params, scales):
            p.grad = (randn(*p.shape) * s).to(p.dtype)
        if case["norm"] == "inf":
            about = max(s * math.sqrt(2 * math.log(1 + p.numel())) for p, s in zip(params, scales))
        else:
            about = math.sqrt(sum(s * s * p.numel() for p, s in zip(params, scales)))
        return {"what": "clip", "params": params, "limit": about * (0.5 if case["clips"] else 2.0), "norm": float(case["norm"])}
    rows, d, v, k = case["rows"], case["d"], case["v"], case["k"]
    weight = 2 * randn(v, d) / math.sqrt(d)
    legal = None
    if case["legal"]:
        # about 30 legal moves to a row; a finished game (one row in 64) has none
        legal = (rand(rows, v) < LEGAL / v) & (rand(rows, 1) >= 1 / 64)
    if case["targets"] == "index":
        index = torch.randint(0, v, (rows,), generator=gen, device=DEV)
        listed_, share = index[:, None], torch.ones(rows, 1, device=DEV)
        index = index.masked_fill(rand(rows) < 1 / 16, -1)              # rows that do not count
        visits = None
    else:
        listed_ = (rand(rows, v) if legal is None else rand(rows, v).masked_fill_(~legal, -1.0)).topk(min(k, v), dim=1)
        share = rand(rows, listed_.indices.shape[1]) ** 3               # a search's visits: few moves take most of them
        share = share.masked_fill(listed_.values < 0, 0.0)
        visits = share / share.sum(1, keepdim=True).clamp_(min=1e-30)
        index = listed_.indices.masked_fill(listed_.values < 0, -1).to(torch.int32)
        listed_, share = listed_.indices, visits
    # normalised activity that has learnt some of it: a row leans to its targets' weights
    x = randn(rows, d)
    lean = 2 * rand(rows, 1)
    top = share.argmax(1)
    x += lean * weight[listed_.gather(1, top[:, None]).squeeze(1)]
    dtype = DTYPES[case["dtype"]]
    return {"what": "loss", "x": x.clamp_(-8, 8).to(dtype), "weight": weight.to(dtype), "bias": (0.1 * randn(v)).to(dtype),
            "index": index, "visits": visits, "legal": legal, "direction": case["direction"],
            # the mean over rows; half precision takes the sum, whose gradients stay clear of its smallest numbers
            "grad_scale": 1.0 if case["dtype"] == "f16" else 1.0 / rows}


def _plain_loss(s):
    x, w = s["x"].float(), s["weight"].float()
    z = x @ w.t() + s["bias"].float()
    if s["legal"] is not None:
        z = torch.where(s["legal"], z, -math.inf)
    index = s["index"].long() if s["visits"] is not None else s["index"].long()[:, None]
    share = s["visits"] if s["visits"] is not None else torch.ones_like(index, dtype=torch.float32)
    spot = index.clamp(min=0)
    out = index < 0
    if s["legal"] is not None:
        out = out | ~s["legal"].gather(1, spot)
    share = torch.where(out, 0.0, share)
    top = z.amax(1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    e = torch.exp(z - top)
    total = e.sum(1, keepdim=True)
    far = total.log() + top - z.gather(1, spot)
    loss = torch.where(out, 0.0, share * far).sum(1)
    if s["direction"] == "loss":
        return loss
    whole = share.sum(1, keepdim=True)
    g = e * torch.where(whole == 0, 0.0, whole / total)
    g = g.scatter_add_(1, spot, -share) * s["grad_scale"]
    return loss, (g @ w).to(s["x"].dtype), (g.t() @ x).to(s["weight"].dtype), g.sum(0).to(s["bias"].dtype)


def _plain_clip(s):
    grads = [p.grad for p in s["params"]]
    if s["norm"] == math.inf:
        norm = torch.stack([g.abs().amax().float() for g in grads]).amax()
    else:
        norm = torch.stack([g.float().square().sum() for g in grads]).sum().sqrt()
    scale = (s["limit"] / (norm + 1e-6)).clamp(max=1.0)
    return norm, *[g.copy_(g.float() * scale) for g in grads]


def run(state):
    if not own:
        return {"loss": _plain_loss, "clip": _plain_clip}[state["what"]](state)
    if state["what"] == "clip":
        from chessfly.clip import clip_grad_norm_
        return clip_grad_norm_(state["params"], state["limit"], state["norm"]), *[p.grad for p in state["params"]]
    from chessfly.readout import Visits, readout_loss, readout_loss_and_grad
    target = state["index"] if state["visits"] is None else Visits(state["index"], state["visits"])
    if state["direction"] == "loss":
        return readout_loss(state["x"], state["weight"], state["bias"], target, legal=state["legal"], reduction="none")
    loss, grads = readout_loss_and_grad(state["x"], state["weight"], state["bias"], target, legal=state["legal"],
                                        grad_scale=state["grad_scale"])
    return loss, *grads


def _exact_loss(s):
    """By autograd, from the targets as distributions over the columns."""
    grads = s["direction"] == "gradient"
    x, w, b = (s[n].double().requires_grad_(grads) for n in ("x", "weight", "bias"))
    rows, v = x.shape[0], w.shape[0]
    target = torch.zeros(rows, v, dtype=torch.float64, device=DEV)
    r, c = (s["index"].view(rows, -1) >= 0).nonzero(as_tuple=True)
    at = s["index"].view(rows, -1)[r, c].long()
    target.index_put_((r, at), s["visits"][r, c].double() if s["visits"] is not None else target.new_ones(()), accumulate=True)
    z = torch.addmm(b, x, w.t())
    if s["legal"] is not None:
        target = target * s["legal"]
        z = z.masked_fill(~s["legal"], -1e300)                          # far below any logit: exp gives 0, without NaN
    loss = -(target * torch.log_softmax(z, 1)).sum(1)
    if not grads:
        return loss
    return loss.detach(), *torch.autograd.grad(loss.sum() * s["grad_scale"], (x, w, b))


def _exact_clip(s):
    grads = [p.grad.double() for p in s["params"]]
    norm = torch.linalg.vector_norm(torch.stack([torch.linalg.vector_norm(g, s["norm"]) for g in grads]), s["norm"])
    return norm, *[g * torch.clamp(s["limit"] / (norm + 1e-6), max=1.0) for g in grads]


def exact(case, seed):
    state = prepare(case, seed)
    return {"loss": _exact_loss, "clip": _exact_clip}[case["what"]](state)


def work(case):
    if case["what"] == "clip":
        sizes, each = [math.prod(s) for s in _shapes(case)], [t.itemsize for t in _types(case)]
        # read once, and written where the norm passes the limit; a product and a sum for each, and the scaling
        return {"bytes": (2 if case["clips"] else 1) * sum(n * b for n, b in zip(sizes, each)), "flops": 3 * sum(sizes)}
    rows, d, v, b = case["rows"], case["d"], case["v"], BYTES[case["dtype"]]
    lists = rows * (8 if case["targets"] == "index" else 8 * case["k"])
    moved = (rows * d + v * d + v) * b + lists + 4 * rows + (rows * v if case["legal"] else 0)
    if case["direction"] == "loss":
        return {"bytes": moved, "flops": 2 * rows * d * v}
    return {"bytes": moved + (rows * d + v * d + v) * b, "flops": 6 * rows * d * v}
