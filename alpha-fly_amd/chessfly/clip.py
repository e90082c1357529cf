"""The norm of all parameters' gradients and clipping by it: `grad_norm` and `clip_grad_norm_`, over fly_clip_gradients.

    norm = sqrt(sum g^2) or max |g|,    g <- g * min(1, limit / (norm + 1e-6))

Arguments as torch.nn.utils.clip_grad_norm_ takes them, but for `foreach`; the norms are 2 and inf, all gradients lie on one device and
each parameter is given once.  Gradients may differ in type (float32, float16, bfloat16) and size; squares are summed in float64.
Gradients of norm below the limit are read and not written.
"""

from __future__ import annotations

import math
from array import array
from collections.abc import Iterable

import torch

from . import _hip

FLOATS = _hip.FLOAT_TYPES


def _dense(g: torch.Tensor) -> bool:
    """Whether g's elements fill its memory without gaps or overlaps, in whatever order."""
    return g.is_contiguous() or torch.ops.aten.is_non_overlapping_and_dense(g)


def _apart(g: torch.Tensor) -> bool:
    """Whether no two elements share memory, of a tensor whose dimensions nest."""
    span = 1
    for stride, size in sorted((st, n) for st, n in zip(g.stride(), g.shape) if n > 1):
        if stride < span:
            return False
        span = stride * (size - 1) + span
    return True


def _gradients(parameters, what: str) -> list[torch.Tensor]:
    if isinstance(parameters, torch.Tensor):
        parameters = (parameters,)
    elif not isinstance(parameters, Iterable):
        raise RuntimeError(f"{what}: parameters must be a tensor or tensors, got {type(parameters).__name__}")
    return [g for p in parameters if (g := p.grad) is not None]


def _run(grads: list[torch.Tensor], limit: float, norm_type: float, what: str) -> torch.Tensor:
    norm_type = float(norm_type)
    if norm_type not in (2.0, math.inf):
        raise RuntimeError(f"{what}: norm_type must be 2 or inf, got {norm_type}")
    if not grads:
        return torch.zeros(())
    n, dev, index = len(grads), grads[0].device, grads[0].get_device()
    if index < 0:
        _hip.require_device(grads[0], what)
    kept, pointers, sizes, types = [], array("Q"), array("q"), array("i")
    for g in grads:
        kind = FLOATS.get(g.dtype)
        if kind is None or g.layout is not torch.strided:
            raise RuntimeError(f"{what}: gradients must be dense float32, float16 or bfloat16, got {g.dtype} {g.layout}")
        if g.get_device() != index:
            raise RuntimeError(f"{what}: gradients must be on one device, got {dev} and {g.device}")
        k = g
        if not _dense(g):
            if limit >= 0 and not _apart(g):
                raise RuntimeError(f"{what}: a gradient's elements overlap in memory")
            k = g.contiguous()
        kept.append(k)
        pointers.append(k.data_ptr())
        sizes.append(k.numel())
        types.append(kind)
    norm = torch.empty((), dtype=torch.float32, device=dev)
    at = [a.buffer_info()[0] for a in (pointers, sizes, types)]      # the arrays outlive the call
    need = _hip.load().fly_clip_workspace(*at[1:], n)
    ws = _hip.workspace(need, dev)
    _hip.call("fly_clip_gradients", index, *at, n, 0 if norm_type == math.inf else 2, limit, norm.data_ptr(),
              ws.data_ptr(), need)
    if limit >= 0:
        for g, k in zip(grads, kept):
            if g is not k:
                g.copy_(k)
        torch.autograd.graph.increment_version(kept)
    return norm


@torch.no_grad()
def grad_norm(parameters, norm_type: float = 2.0) -> torch.Tensor:
    """The norm (2 or inf) of the parameters' gradients together, as a float32 tensor without dimensions; parameters without a
    gradient are left out."""
    return _run(_gradients(parameters, "grad_norm"), -1.0, norm_type, "grad_norm")


@torch.no_grad()
def clip_grad_norm_(parameters, max_norm: float, norm_type: float = 2.0, error_if_nonfinite: bool = False) -> torch.Tensor:
    """Scales the parameters' gradients in place so that their norm together is at most max_norm, and returns the norm that they
    had, float32 on their device.  A parameter may be given once; gradients must not share memory.  A NaN in any gradient makes
    all of them NaN, as in torch, unless error_if_nonfinite, which waits for the norm and raises before anything is scaled."""
    what, max_norm = "clip_grad_norm_", float(max_norm)
    if not max_norm >= 0:
        raise RuntimeError(f"{what}: max_norm must be at least 0, got {max_norm}")
    grads = _gradients(parameters, what)
    if error_if_nonfinite and grads:
        norm = _run(grads, -1.0, norm_type, what)
        if not math.isfinite(norm):
            raise RuntimeError(f"{what}: the gradients' norm is {float(norm)}")
    return _run(grads, max_norm, norm_type, what)
