"""Softmax cross entropy of a read-out, without keeping its logits: `readout_loss` and `readout_loss_and_grad`, over
fly_readout_loss.

    z_r  = x_r W^T + b over the legal columns
    loss = sum_j a_rj (log sum exp z_r - z_r,t_rj)      a list of columns t with weights a (visits), or one column with weight 1

and its gradients by x, W and b.  The loss alone keeps no logits; with gradients those of a piece of rows at a time are kept with their
gradients, 12 bytes of a float32 logit and 6 of a 16-bit one, 4 GiB at most, beside both operands laid out for the matrix cores.  Past
that size memory no longer grows with rows times columns; below it, a call takes more than float32 logits alone would.

Sums are float32 whatever the type, and results do not depend on scheduling.  From some dozens of rows on float32 operands are
multiplied in 22 bits, and with 16-bit ones the logits' gradient is rounded to their type before its products (include/flyeval.h): the
gradients then err by 1.1 to 1.4 times what rounding them to the type does, in the norm.  float32 operands avoid that.  No counterpart in the
reference, whose training takes torch's softmax over all logits.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _hip

FLOATS = _hip.FLOAT_TYPES
INDEX = {torch.int32: 4, torch.int64: 5}
MOST_LISTED = 1024


class Visits(NamedTuple):
    """A row's targets: index (rows, k) int32 or int64 (negative: none) and weight (rows, k) float32, as a search's visits give
    them.  Weights need not add to 1; those of a column listed twice add up."""
    index: torch.Tensor
    weight: torch.Tensor


class ReadoutGrads(NamedTuple):
    """Gradients by the read-out's inputs, weight and bias (None without one), each of its tensor's type."""
    x: torch.Tensor | None
    weight: torch.Tensor | None
    bias: torch.Tensor | None


class _Call(NamedTuple):
    """Checked arguments: the tensors as the kernel takes them, and the distances of their rows."""
    x: torch.Tensor
    ldx: int
    weight: torch.Tensor
    ldw: int
    bias: torch.Tensor | None
    legal: torch.Tensor | None
    ldl: int
    index: torch.Tensor
    share: torch.Tensor | None


def _checked(x, weight, bias, target, legal, what: str) -> _Call:
    _hip.require_device(x, what)
    dev = x.device
    if x.dim() != 2 or weight.dim() != 2 or x.shape[1] != weight.shape[1] or weight.device != dev:
        raise RuntimeError(f"{what}: x and weight must be (rows, d) and (columns, d) on one device, got {tuple(x.shape)} on {dev} "
                           f"and {tuple(weight.shape)} on {weight.device}")
    if x.dtype not in FLOATS or weight.dtype != x.dtype:
        raise RuntimeError(f"{what}: x and weight must both be float32, float16 or bfloat16, got {x.dtype} and {weight.dtype}")
    rows, cols = x.shape[0], weight.shape[0]
    if bias is not None:
        if bias.dtype not in (x.dtype, torch.float32) or bias.shape != (cols,) or bias.device != dev:
            raise RuntimeError(f"{what}: bias must be {x.dtype} or float32 of shape ({cols},) on {dev}, got {bias.dtype} "
                               f"{tuple(bias.shape)} on {bias.device}")
        bias = bias.contiguous()
    share = None
    if isinstance(target, torch.Tensor):
        index, shape = target, (rows,)
    else:
        index, share = target
        shape = (rows, share.shape[-1] if share.dim() else 0)
        if share.dtype != torch.float32 or share.shape != shape or share.device != dev or not 1 <= shape[1] <= MOST_LISTED:
            raise RuntimeError(f"{what}: the targets' weights must be float32 of shape ({rows}, 1..{MOST_LISTED}) on {dev}, got "
                               f"{share.dtype} {tuple(share.shape)} on {share.device}")
        share = share.contiguous()
    if index.dtype not in INDEX or index.shape != shape or index.device != dev:
        raise RuntimeError(f"{what}: the targets must be int32 or int64 of shape {shape} on {dev}, got {index.dtype} "
                           f"{tuple(index.shape)} on {index.device}")
    ldl = 0
    if legal is not None:
        if legal.dtype not in (torch.bool, torch.uint8) or legal.shape != (rows, cols) or legal.device != dev:
            raise RuntimeError(f"{what}: legal must be bool of shape ({rows}, {cols}) on {dev}, got {legal.dtype} "
                               f"{tuple(legal.shape)} on {legal.device}")
        legal, ldl = _hip.row_major(legal)
    x, ldx = _hip.row_major(x)
    weight, ldw = _hip.row_major(weight)
    return _Call(x, ldx, weight, ldw, bias, legal, ldl, index.contiguous(), share)


def _run(c: _Call, loss, row_scale, grad_scale: float, want: tuple[bool, bool, bool]) -> ReadoutGrads:
    (rows, d), cols, dev = c.x.shape, c.weight.shape[0], c.x.device
    gx = torch.empty(rows, d, dtype=c.x.dtype, device=dev) if want[0] else None
    gw = torch.empty(cols, d, dtype=c.x.dtype, device=dev) if want[1] else None
    gb = torch.empty(cols, dtype=c.bias.dtype, device=dev) if want[2] else None
    kind, wanted = FLOATS[c.x.dtype], want[0] + 2 * want[1] + 4 * want[2]
    k = c.share.shape[1] if c.share is not None else 1
    need = _hip.load().fly_readout_loss_workspace(kind, rows, d, cols, k, wanted)
    ws = _hip.workspace(need, dev)
    _hip.call("fly_readout_loss", dev.index, c.x.data_ptr(), kind, c.ldx, rows, d, c.weight.data_ptr(), c.ldw, cols,
              _hip.ptr(c.bias), FLOATS[c.bias.dtype] if c.bias is not None else 0, _hip.ptr(c.legal), c.ldl,
              c.index.data_ptr(), INDEX[c.index.dtype], _hip.ptr(c.share), k,
              _hip.ptr(loss), _hip.ptr(row_scale), grad_scale, _hip.ptr(gx), d, _hip.ptr(gw), d, _hip.ptr(gb), ws.data_ptr(),
              need)
    return ReadoutGrads(gx, gw, gb)


def readout_loss_and_grad(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None, target, grad_scale: float = 1.0,
                          legal: torch.Tensor | None = None,
                          row_scale: torch.Tensor | None = None) -> tuple[torch.Tensor, ReadoutGrads]:
    """The loss of each row (float32) and, in the same pass, the gradients of grad_scale * sum(row_scale * loss) by x, weight and
    bias (grad_scale = 1 / rows: of the mean).  A row whose row_scale is 0 reaches no gradient, whatever it holds.  For training loops;
    autograd does not follow the results."""
    what = "readout_loss_and_grad"
    c = _checked(x.detach(), weight.detach(), bias.detach() if bias is not None else None, target, legal, what)
    rows = c.x.shape[0]
    if row_scale is not None:
        if row_scale.dtype != torch.float32 or row_scale.shape != (rows,) or row_scale.device != c.x.device:
            raise RuntimeError(f"{what}: row_scale must be float32 of shape ({rows},) on {c.x.device}, "
                               f"got {row_scale.dtype} {tuple(row_scale.shape)} on {row_scale.device}")
        row_scale = row_scale.contiguous()
    loss = torch.empty(rows, dtype=torch.float32, device=c.x.device)
    return loss, _run(c, loss, row_scale, grad_scale, (True, True, bias is not None))


class _ReadoutLoss(torch.autograd.Function):
    """Rows' losses; the backward runs the whole call again for the gradients that are needed, scaled by the rows' upstream
    gradients, so nothing but the inputs is kept between the two."""

    @staticmethod
    def forward(ctx, x, weight, bias, legal, index, share, ldx, ldw, ldl):
        c = _Call(x, ldx, weight, ldw, bias, legal, ldl, index, share)
        loss = torch.empty(x.shape[0], dtype=torch.float32, device=x.device)
        _run(c, loss, None, 1.0, (False, False, False))
        ctx.save_for_backward(x, weight, bias, legal, index, share)
        ctx.rest = ldx, ldw, ldl
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, up):
        x, weight, bias, legal, index, share = ctx.saved_tensors
        ldx, ldw, ldl = ctx.rest
        if not any(ctx.needs_input_grad[:3]):
            return (None,) * 9
        c = _Call(x, ldx, weight, ldw, bias, legal, ldl, index, share)
        grads = _run(c, None, up.float().contiguous(), 1.0, ctx.needs_input_grad[:3])
        return (*grads,) + (None,) * 6


def readout_loss(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None, target, legal: torch.Tensor | None = None,
                 reduction: str = "mean") -> torch.Tensor:
    """Softmax cross entropy of x (rows, d) W^T + b against `target`: Visits, or one column a row (rows) int32 or int64 (negative:
    the row is left out).  x and weight (columns, d) float32, float16 or bfloat16, bias of that type or float32; legal (rows,
    columns) bool hides columns.  Differentiable once by x, weight and bias; a backward pass to the targets' weights raises.
    reduction: "mean" or "sum" over all rows, or "none" (rows) float32.

    A target that `legal` hides, or of weight 0, is left out; a row with none left has loss and gradients 0, whatever it holds, and one
    whose loss gets an upstream gradient of 0 reaches no gradient.  A target past the columns makes its row NaN."""
    what = "readout_loss"
    if reduction not in ("mean", "sum", "none"):
        raise RuntimeError(f"{what}: reduction must be mean, sum or none, got {reduction!r}")
    c = _checked(x, weight, bias, target, legal, what)
    share = c.share
    if share is not None and _hip.tracked(share):
        share = _hip.undifferentiated(f"{what} by its targets' weights", c.share.clone, c.share)
    if any(t is not None and _hip.tracked(t) for t in (x, weight, bias, share)):
        nodes = _hip.held_leaves(what, x, weight, bias)  # noqa: F841  (alive until the graph has them)
        loss = _ReadoutLoss.apply(c.x, c.weight, c.bias, c.legal, c.index, share, c.ldx, c.ldw, c.ldl)
    else:
        loss = torch.empty(c.x.shape[0], dtype=torch.float32, device=c.x.device)
        _run(c, loss, None, 1.0, (False, False, False))
    return loss if reduction == "none" else loss.mean() if reduction == "mean" else loss.sum()
