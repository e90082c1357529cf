"""Distillation from a teacher's top logits: `top_logits`, `distill_loss`, `distill_loss_and_grad`, over fly_top_logits
and fly_distill, and `label`, which runs a teacher.

A teacher labels positions once: of each row of its logits the k largest are kept, and the log-sum-exp of the rest, which
is what a replay buffer has to hold.  A student then learns from that list:

    p, p_t = softmax of (values / T, tail)                     the listed moves, and one class for all others
    q      = softmax of (logits / T) over the visible moves,   q_t = its sum over the moves not listed
    loss   = T^2 (sum_S p log(p / q) + p_t log(p_t / q_t))

Rows are independent, sums are float32 whatever the logits' type, and results do not depend on scheduling.
No counterpart in the reference, whose training takes visit counts over all moves.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _hip

FLOATS = _hip.FLOAT_TYPES
MOST_LISTED = 256      # no chess position has over 218 legal moves


class TopLogits(NamedTuple):
    """A teacher's list: values (rows, k) float32 in falling order, index (rows, k) int32 (-1: no such move), and tail
    (rows) float32, the log-sum-exp at the temperature of what is not listed (None: the list is all there is)."""
    values: torch.Tensor
    index: torch.Tensor
    tail: torch.Tensor | None = None


def _logits(logits: torch.Tensor, what: str) -> tuple[torch.Tensor, int]:
    _hip.require_device(logits, what)
    if logits.dim() != 2 or logits.shape[1] < 1:
        raise RuntimeError(f"{what}: logits must be (rows, columns), got {tuple(logits.shape)}")
    if logits.dtype not in FLOATS:
        raise RuntimeError(f"{what}: logits must be float32, float16 or bfloat16, got {logits.dtype}")
    return _hip.row_major(logits)


def _legal(legal: torch.Tensor | None, logits: torch.Tensor, what: str) -> tuple[torch.Tensor | None, int]:
    if legal is None:
        return None, 0
    if legal.dtype not in (torch.bool, torch.uint8) or legal.shape != logits.shape or legal.device != logits.device:
        raise RuntimeError(f"{what}: legal must be bool of shape {tuple(logits.shape)} on {logits.device}, "
                           f"got {legal.dtype} {tuple(legal.shape)} on {legal.device}")
    return _hip.row_major(legal)


def top_logits(logits: torch.Tensor, k: int, temperature: float = 1.0, legal: torch.Tensor | None = None,
               tail: bool = True) -> TopLogits:
    """The k (1 to 256) largest logits of each row over the legal columns, the lower column first among equals, and the
    log-sum-exp of the others.  Rows with fewer legal columns (a column at -inf is none) end in values -inf and index -1;
    a tail of nothing is -inf.  Not differentiable: a backward pass through the values or the tail raises."""
    if _hip.tracked(logits):
        return TopLogits(*_hip.undifferentiated(
            "top_logits", lambda: tuple(top_logits(logits, k, temperature, legal, tail)), logits))
    logits, ld = _logits(logits, "top_logits")
    legal, ld_legal = _legal(legal, logits, "top_logits")
    rows, cols = logits.shape
    dev = logits.device
    k = int(k)
    if not 1 <= k <= MOST_LISTED:
        raise RuntimeError(f"top_logits: k must lie in 1..{MOST_LISTED}, got {k}")
    values = torch.empty(rows, k, dtype=torch.float32, device=dev)
    index = torch.empty(rows, k, dtype=torch.int32, device=dev)
    rest = torch.empty(rows, dtype=torch.float32, device=dev) if tail else None
    _hip.call("fly_top_logits", dev.index, logits.data_ptr(), FLOATS[logits.dtype], ld, rows, cols, _hip.ptr(legal),
              ld_legal, k, temperature, values.data_ptr(), index.data_ptr(), _hip.ptr(rest))
    return TopLogits(values, index, rest)


def _teacher(teacher, logits: torch.Tensor, what: str) -> TopLogits:
    values, index, tail = teacher = teacher if type(teacher) is TopLogits else TopLogits(*teacher)
    rows, dev = logits.shape[0], logits.device
    if not (values.dtype is torch.float32 and index.dtype is torch.int32 and values.dim() == 2 and values.shape[0] == rows
            and values.device == dev and index.device == dev
            and (tail is None or (tail.dtype is torch.float32 and tail.shape == (rows,) and tail.device == dev))):
        raise RuntimeError(f"{what}: the teacher's values, index and tail must be float32, int32 and float32 (or None) with "
                           f"{rows} rows on {dev}, got " + ", ".join(
                               "None" if t is None else f"{t.dtype} {tuple(t.shape)} on {t.device}" for t in teacher))
    if values.shape != index.shape or not 1 <= values.shape[1] <= MOST_LISTED:
        raise RuntimeError(f"{what}: the teacher's values and index must be alike, (rows, 1..{MOST_LISTED}), got "
                           f"{tuple(values.shape)} and {tuple(index.shape)}")
    if values.is_contiguous() and index.is_contiguous() and (tail is None or tail.is_contiguous()):
        return teacher
    return TopLogits(*(t.contiguous() if t is not None else None for t in teacher))


def _run(logits, ld, values, index, tail, temperature, legal, ld_legal, loss, grad, row_scale, grad_scale) -> None:
    rows, cols = logits.shape
    _hip.call("fly_distill", logits.device.index, logits.data_ptr(), FLOATS[logits.dtype], ld, rows, cols,
              _hip.ptr(legal), ld_legal, values.data_ptr(), index.data_ptr(), _hip.ptr(tail), values.shape[1], temperature,
              _hip.ptr(loss), _hip.ptr(grad), cols, _hip.ptr(row_scale), grad_scale)


def distill_loss_and_grad(logits: torch.Tensor, teacher: TopLogits, temperature: float = 1.0,
                          legal: torch.Tensor | None = None, grad_scale: float = 1.0,
                          row_scale: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The loss of each row (float32) and, in the same pass, grad_scale * row_scale * dloss/dlogits in the logits' type
    (grad_scale = 1 / rows: the gradient of the mean).  For training loops: `logits.backward(grad)`; autograd does not follow
    the two results themselves."""
    what = "distill_loss_and_grad"
    logits, ld = _logits(logits, what)
    legal, ld_legal = _legal(legal, logits, what)
    teacher = _teacher(teacher, logits, what)
    rows, cols = logits.shape
    if row_scale is not None:
        if row_scale.dtype != torch.float32 or row_scale.shape != (rows,) or row_scale.device != logits.device:
            raise RuntimeError(f"{what}: row_scale must be float32 of shape ({rows},) on {logits.device}, "
                               f"got {row_scale.dtype} {tuple(row_scale.shape)} on {row_scale.device}")
        row_scale = row_scale.contiguous()
    loss = torch.empty(rows, dtype=torch.float32, device=logits.device)
    grad = torch.empty(rows, cols, dtype=logits.dtype, device=logits.device)
    _run(logits, ld, *teacher, temperature, legal, ld_legal, loss, grad, row_scale, grad_scale)
    return loss, grad


class _DistillLoss(torch.autograd.Function):
    """Rows' losses; the backward is the kernel's gradient pass over the saved logits, scaled by the rows' upstream
    gradients."""

    @staticmethod
    def forward(ctx, logits, ld, values, index, tail, temperature, legal, ld_legal):
        loss = torch.empty(logits.shape[0], dtype=torch.float32, device=logits.device)
        _run(logits, ld, values, index, tail, temperature, legal, ld_legal, loss, None, None, 1.0)
        ctx.save_for_backward(logits, values, index, tail, legal)
        ctx.rest = ld, temperature, ld_legal
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, up):
        logits, values, index, tail, legal = ctx.saved_tensors
        grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        ld, temperature, ld_legal = ctx.rest
        _run(logits, ld, values, index, tail, temperature, legal, ld_legal, None, grad, up.float().contiguous(), 1.0)
        return (grad,) + (None,) * 7


def distill_loss(logits: torch.Tensor, teacher: TopLogits, temperature: float = 1.0,
                 legal: torch.Tensor | None = None, reduction: str = "mean") -> torch.Tensor:
    """The student's loss against a teacher's list, differentiable once by `logits` (the teacher's tensors get no gradient).
    reduction: "mean" or "sum" over rows, or "none" (rows) float32.

    A row without a listed legal move (index -1, or a move that `legal` hides), or whose student sees no move, has loss
    and gradient 0.  The tail is left out where the student has no move outside the list.  A repeated index, or one past
    the columns, makes its row NaN."""
    if reduction not in ("mean", "sum", "none"):
        raise RuntimeError(f"distill_loss: reduction must be mean, sum or none, got {reduction!r}")
    logits, ld = _logits(logits, "distill_loss")
    legal, ld_legal = _legal(legal, logits, "distill_loss")
    teacher = _teacher(teacher, logits, "distill_loss")
    if _hip.tracked(logits):      # in forward mode torch says that there is no such derivative
        loss = _DistillLoss.apply(logits, ld, *(t.detach() if t is not None else None for t in teacher), temperature, legal,
                                  ld_legal)
    else:
        loss = torch.empty(logits.shape[0], dtype=torch.float32, device=logits.device)
        _run(logits, ld, *teacher, temperature, legal, ld_legal, loss, None, None, 1.0)
    return loss if reduction == "none" else loss.mean() if reduction == "mean" else loss.sum()


@torch.no_grad()
def label(teacher, x: torch.Tensor, k: int, temperature: float = 1.0,
          legal: torch.Tensor | None = None) -> tuple[TopLogits, torch.Tensor]:
    """What a replay buffer keeps of a teacher network (in eval mode; head_dtype int8 does for it) on boards x: its k best
    legal moves with the rest's log-sum-exp, and its WDL logits."""
    if teacher.training:
        raise RuntimeError("label: the teacher must be in eval mode")
    logits, wdl = teacher(x)
    return top_logits(logits, k, temperature, legal), wdl
