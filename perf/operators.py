"""The 8-bit and distillation operators, as cases that can be timed and checked.

A teacher labels positions: its read-out runs as a matrix product in 8-bit integers, and of each row of logits the
largest are kept, with the log-sum-exp of the rest.  A student then learns from them.

Kinds of work ("what"):
* linear   Int8Linear: rows of activity to 8 bits with a scale for each row, times a weight held in 8 bits with a scale
           for each channel, plus the bias.
* top      top_logits: the k largest visible logits of each row, ties to the lower column, and the log-sum-exp of the
           others at the temperature.
* distill  the student's loss against a teacher's list, the Kullback-Leibler divergence over the listed columns and one
           bucket for the rest, and its gradient with respect to the student's logits ("direction": "loss" or
           "gradient", which returns both).
"""

from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "alpha-fly_amd"))

own = False

DEV = "cuda:0"
N_MOVES, N_OUT = 4168, 2333          # the policy's moves, the output neurons that it reads
N_BOARD, N_SENSORY = 838, 17937      # the board's features, the sensory neurons that they drive
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
LEGAL = 30                           # legal moves of a chess position, about


def listed():
    return [
        # one position's policy read-out: a game against the engine
        {"name": "read-out, one position", "what": "linear", "rows": 1, "k": N_OUT, "n": N_MOVES, "dtype": "f32",
         "out": "f32"},
        # the same for a search with a few games left
        {"name": "read-out, handful", "what": "linear", "rows": 21, "k": N_OUT, "n": N_MOVES, "dtype": "f32",
         "out": "f32"},
        # one leaf of each of 1,120 games
        {"name": "read-out, self-play", "what": "linear", "rows": 1120, "k": N_OUT, "n": N_MOVES, "dtype": "f32",
         "out": "f32"},
        # the boards' map onto the sensory neurons, half precision in and out, an odd batch and odd sizes
        {"name": "board map", "what": "linear", "rows": 517, "k": N_BOARD, "n": N_SENSORY, "dtype": "f16",
         "out": "f16"},
        # a part of a replay buffer labelled by the teacher
        {"name": "read-out, labelling", "what": "linear", "rows": 16384, "k": N_OUT, "n": N_MOVES, "dtype": "f32",
         "out": "f16"},
        # every legal move of one position (no position has over 218)
        {"name": "one position's moves", "what": "top", "rows": 1, "v": N_MOVES, "k": 218, "dtype": "f32",
         "legal": True, "temperature": 1.0},
        # the labels of a self-play batch over all moves
        {"name": "self-play's labels", "what": "top", "rows": 1120, "v": N_MOVES, "k": 32, "dtype": "f32",
         "legal": False, "temperature": 1.0},
        # labels over a vocabulary of words
        {"name": "labels, vocabulary", "what": "top", "rows": 4096, "v": 32000, "k": 64, "dtype": "bf16",
         "legal": False, "temperature": 2.0},
        # a training step's batch on legal moves
        {"name": "training batch", "what": "distill", "rows": 256, "v": N_MOVES, "k": 32, "dtype": "f32",
         "legal": True, "tail": True, "temperature": 1.0, "direction": "gradient"},
        # the loss alone on held-out positions
        {"name": "held-out positions", "what": "distill", "rows": 1120, "v": N_MOVES, "k": 24, "dtype": "f32",
         "legal": False, "tail": True, "temperature": 1.5, "direction": "loss"},
        # a large batch of half-precision logits
        {"name": "large batch", "what": "distill", "rows": 16384, "v": N_MOVES, "k": 32, "dtype": "f16",
         "legal": False, "tail": True, "temperature": 2.0, "direction": "gradient"},
        # a vocabulary of words of odd size, the teacher's list alone
        {"name": "vocabulary", "what": "distill", "rows": 2048, "v": 50257, "k": 64, "dtype": "bf16",
         "legal": False, "tail": False, "temperature": 1.0, "direction": "gradient"},
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    what = rng.choice(["linear", "top", "distill"])
    if what == "linear":
        k, n = rng.choice([(N_OUT, N_MOVES), (N_BOARD, N_SENSORY),
                           (_log_uniform(rng, 64, 5000), _log_uniform(rng, 64, 20000))])
        # no more work than the labelling case
        rows = _log_uniform(rng, 1, max(1, min(16384, 16384 * N_OUT * N_MOVES // (k * n), 60_000_000 // n)))
        return {"what": what, "rows": rows, "k": k, "n": n, "dtype": rng.choice(list(DTYPES)),
                "out": rng.choice(list(DTYPES))}
    v = rng.choice([N_MOVES, _log_uniform(rng, 300, 50257)])
    dtype = rng.choice(list(DTYPES))
    rows = _log_uniform(rng, 1, max(1, min(16384, 100_000_000 // (v * (BYTES[dtype] // 2)))))
    legal = v == N_MOVES and rng.random() < 0.5
    case = {"what": what, "rows": rows, "v": v, "k": _log_uniform(rng, 1, 256), "dtype": dtype, "legal": legal,
            "temperature": rng.choice([0.5, 1.0, 2.0, 4.0])}
    if what == "distill":
        case["tail"] = rng.random() < 0.5
        case["direction"] = rng.choice(["loss", "gradient"])
    return case


def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) & 0x7FFFFFFF)


def _legal(rows, v, gen):
    """About 30 visible moves to a row; a finished game (one row in 64) has none."""
    legal = torch.rand(rows, v, generator=gen, device=DEV) < LEGAL / v
    over = torch.rand(rows, 1, generator=gen, device=DEV) < 1 / 64
    return legal & ~over


def prepare(case, seed):
    gen = _generator(seed)
    rows = case["rows"]
    randn = lambda *s: torch.randn(*s, generator=gen, device=DEV)
    if case["what"] == "linear":
        k, n = case["k"], case["n"]
        w = randn(n, k) / math.sqrt(k)
        scale = w.abs().amax(1) / 127
        state = {"x": randn(rows, k).clamp_(-8, 8).to(DTYPES[case["dtype"]]),   # normalised activity
                 "weight": torch.round(w / scale[:, None]).clamp_(-127, 127).to(torch.int8),
                 "scale": scale, "bias": 0.1 * randn(n), "out": DTYPES[case["out"]]}
        if own:
            from chessfly.int8 import Int8Linear
            state["plan"] = Int8Linear(state["weight"], state["scale"], state["bias"])
        return {"what": "linear", **state}
    v, k = case["v"], case["k"]
    legal = _legal(rows, v, gen) if case["legal"] else None
    logits = 3 * randn(rows, v)
    state = {"what": case["what"], "k": k, "temperature": case["temperature"], "legal": legal,
             "logits": logits.to(DTYPES[case["dtype"]])}
    if case["what"] == "distill":
        teacher = logits + randn(rows, v)
        if legal is not None:
            teacher.masked_fill_(~legal, -math.inf)
        kk = min(k, v)
        values, index = teacher.topk(kk, dim=1)
        rest = (teacher / case["temperature"]).scatter(1, index, -math.inf)
        state["tail"] = torch.logsumexp(rest, 1) if case["tail"] else None
        none = values == -math.inf
        state["values"] = values.contiguous()
        state["index"] = index.masked_fill(none, -1).to(torch.int32)
        state["direction"] = case["direction"]
        # the mean over rows; half precision takes the sum, whose gradients stay clear of its smallest numbers
        state["grad_scale"] = 1.0 if case["dtype"] == "f16" else 1.0 / rows
    return state


def _plain_linear(s):
    x = s["x"].float()
    top = x.abs().amax(1, keepdim=True)
    q = torch.round(x * (torch.full_like(top, 127.0) / top))
    acc = q @ s["weight"].float().t()
    row = top / torch.full_like(top, 127.0)
    return (acc * (row * s["scale"]) + s["bias"]).to(s["out"])


def _log_sum_exp(z):
    """log sum exp over the last dimension; -inf for a row of nothing but -inf."""
    top = z.amax(-1, keepdim=True)
    base = torch.where(top == -math.inf, torch.zeros_like(top), top)
    return (torch.exp(z - base).sum(-1, keepdim=True).log() + base).squeeze(-1)


def _plain_top(s):
    z, k = s["logits"].float(), s["k"]
    if s["legal"] is not None:
        z = z.masked_fill(~s["legal"], -math.inf)
    values, index = torch.sort(z, dim=1, descending=True, stable=True)
    rest = _log_sum_exp(values[:, k:] * (1.0 / s["temperature"])) if k < z.shape[1] else z.new_full(z.shape[:1], -math.inf)
    pad = max(0, k - z.shape[1])
    values = torch.nn.functional.pad(values[:, :k], (0, pad), value=-math.inf)
    index = torch.nn.functional.pad(index[:, :k], (0, pad), value=-1)
    return values, index.masked_fill(values == -math.inf, -1).to(torch.int32), rest


def _plain_distill(s):
    t, v = s["temperature"], s["logits"].shape[1]
    z = s["logits"].float() * (1.0 / t)
    if s["legal"] is not None:
        z = z.masked_fill(~s["legal"], -math.inf)
    pad = s["index"] < 0
    index = torch.where(pad, 0, s["index"]).long()
    # listed columns; padding goes to a column of its own behind the last
    spot = torch.where(pad, v, s["index"]).long()
    listed_ = torch.zeros(z.shape[0], v + 1, dtype=torch.bool, device=z.device).scatter_(1, spot, True)[:, :v]
    rest = _log_sum_exp(z.masked_fill(listed_, -math.inf))                       # the student's bucket
    zs = z.gather(1, index).masked_fill(pad, -math.inf)
    lse = _log_sum_exp(torch.cat([zs, rest[:, None]], 1))
    a = (s["values"] * (1.0 / t)).masked_fill(pad, -math.inf)                    # the teacher's list
    tail = s["tail"] if s["tail"] is not None else torch.full_like(rest, -math.inf)
    tail = torch.where(rest == -math.inf, -math.inf, tail)
    total = _log_sum_exp(torch.cat([a, tail[:, None]], 1))
    some = (total > -math.inf) & (lse > -math.inf)
    base, total = torch.where(some, lse, 0.0)[:, None], torch.where(some, total, 0.0)[:, None]
    logp = torch.cat([a, tail[:, None]], 1) - total
    logq = torch.cat([zs, rest[:, None]], 1) - base
    p, q = torch.exp(logp), torch.exp(logq)
    # sum p log(p/q), with -p + q in each term: they add to nothing, and an error of a log-sum-exp cancels
    d = torch.where(p > 0, logp - logq, 0.0)
    term = torch.where(d.abs() < 0.5, p * (d + torch.expm1(-d)), p * d - p + q)
    loss = torch.where(some, torch.where(p > 0, term, q).sum(1) * (t * t), 0.0)
    if s["direction"] == "loss":
        return loss
    scale = torch.where(some, t * s["grad_scale"], 0.0)[:, None]
    shift = torch.where(rest == -math.inf, 0.0, rest)[:, None]
    grad = torch.exp(z.masked_fill(listed_, -math.inf) - shift) * ((q[:, -1:] - p[:, -1:]) * scale)
    grad = torch.cat([grad, torch.zeros_like(grad[:, :1])], 1).scatter_(1, spot, (q[:, :-1] - p[:, :-1]) * scale)
    return loss, grad[:, :v].to(s["logits"].dtype)


def run(state):
    what = state["what"]
    if not own:
        return {"linear": _plain_linear, "top": _plain_top, "distill": _plain_distill}[what](state)
    if what == "linear":
        return state["plan"](state["x"], out_dtype=state["out"])
    from chessfly import distill
    if what == "top":
        return tuple(distill.top_logits(state["logits"], state["k"], temperature=state["temperature"],
                                        legal=state["legal"]))
    teacher = distill.TopLogits(state["values"], state["index"], state["tail"])
    if state["direction"] == "loss":
        return distill.distill_loss(state["logits"], teacher, temperature=state["temperature"], legal=state["legal"],
                                    reduction="none")
    return distill.distill_loss_and_grad(state["logits"], teacher, temperature=state["temperature"],
                                         legal=state["legal"], grad_scale=state["grad_scale"])


def _exact_linear(s):
    """The quantisation in the float32 arithmetic that defines it, on the host; the integer sums and scales in 64 bits."""
    x = s["x"].float().cpu().numpy()
    top = np.abs(x).max(1, keepdims=True)
    q = np.rint(x * (np.float32(127) / top)).astype(np.float64)
    row = (top / np.float32(127)).astype(np.float64)
    to = lambda a: torch.from_numpy(a).to(DEV)
    acc = to(q) @ s["weight"].double().t()
    return acc * to(row) * s["scale"].double() + s["bias"].double()


def _exact_top(s):
    z = s["logits"].double()
    if s["legal"] is not None:
        z = torch.where(s["legal"], z, -math.inf)
    k = min(s["k"], z.shape[1])
    best = z.topk(k, dim=1).values
    out = z.new_full((z.shape[0], s["k"]), -math.inf)
    out[:, :k] = best
    # of the columns that equal the last value listed, the list holds the first few
    last = best[:, -1:]
    room = k - (z > last).sum(1, keepdim=True)
    ties = z == last
    kept = (z > last) | (ties & (ties.cumsum(1) <= room))
    return out, None, torch.logsumexp(torch.where(kept, -math.inf, z / s["temperature"]), 1)


def _exact_distill(s):
    """The loss as a divergence of two distributions over the columns' classes, and its gradient by autograd."""
    t = float(s["temperature"])
    z = s["logits"].double().requires_grad_(s["direction"] == "gradient")
    rows, v = z.shape
    seen = s["legal"] if s["legal"] is not None else torch.ones(rows, v, dtype=torch.bool, device=DEV)
    teacher = torch.full((rows, v), -math.inf, dtype=torch.float64, device=DEV)
    r, c = (s["index"] >= 0).nonzero(as_tuple=True)
    teacher[r, s["index"][r, c].long()] = s["values"][r, c].double() / t
    on = teacher > -math.inf
    outside = seen & ~on
    has_rest, row = outside.any(1), on.any(1) | outside.any(1)
    tail = torch.where(has_rest, s["tail"].double(), -math.inf) if s["tail"] is not None else z.new_full((rows,), -math.inf)
    row = row & (torch.logaddexp(torch.logsumexp(teacher, 1), tail) > -math.inf)
    classes = torch.cat([teacher, tail.detach()[:, None]], 1)
    classes = torch.where(row[:, None], classes, 0.0)
    p = classes.softmax(1)
    zt = torch.where(seen, z / t, -1e300)                       # far below any logit: exp gives 0, without NaN
    logq = torch.log_softmax(zt, 1)
    rest = torch.logsumexp(torch.where(outside, logq, -1e300), 1)
    logq = torch.cat([torch.where(on, logq, 0.0), torch.where(has_rest, rest, 0.0)[:, None]], 1)
    term = torch.special.xlogy(p, p) - p * logq
    loss = t * t * torch.where(row[:, None], term, 0.0).sum(1)
    if s["direction"] == "loss":
        return loss
    (grad,) = torch.autograd.grad(loss.sum() * s["grad_scale"], z)
    return loss.detach(), grad


def exact(case, seed):
    state = prepare(case, seed)
    return {"linear": _exact_linear, "top": _exact_top, "distill": _exact_distill}[case["what"]](state)


def work(case):
    rows = case["rows"]
    if case["what"] == "linear":
        k, n = case["k"], case["n"]
        return {"bytes": rows * k * BYTES[case["dtype"]] + n * k + 8 * n + rows * n * BYTES[case["out"]],
                "flops": 2 * rows * k * n}
    v, k = case["v"], case["k"]
    row = v * BYTES[case["dtype"]] + (v if case["legal"] else 0) + 8 * k + 4
    if case["what"] == "distill" and case["direction"] == "gradient":
        row += v * BYTES[case["dtype"]]
    # a scale, a comparison with the largest, an exponential and a sum for each logit, and as much for its gradient
    per = 8 if case["what"] == "distill" and case["direction"] == "gradient" else 4
    return {"bytes": rows * row, "flops": rows * v * per}
