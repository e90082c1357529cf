"""Dense maps held in 8 bits: `quantize_rows` and `Int8Linear`, over fly_quantize_rows and fly_int8_*.

    s_m = max_k |x_mk| / 127,   q_mk = rint(x_mk * (127 / max_k |x_mk|))          a scale for each token
    y_mn = (sum_k q_mk w_nk) (s_m t_n) + b_n                                      and for each channel

The sums are exact in int32; the scales and the bias are applied in float32 and the result rounds once to `out_dtype`.
A token that holds an infinity or NaN has NaN outputs; one of zeros gives the bias.  No counterpart in the reference.
"""

from __future__ import annotations

import ctypes

import torch

from . import _hip

FLOATS = _hip.FLOAT_TYPES


def _rows(x: torch.Tensor, what: str) -> tuple[torch.Tensor, int]:
    _hip.require_device(x, what)
    if x.dim() != 2:
        raise RuntimeError(f"{what}: x must have two dimensions, got {tuple(x.shape)}")
    return _hip.row_major(x)


def quantize_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x (rows, columns) float32, float16 or bfloat16 -> int8 values (rows, columns) and float32 scales (rows).  Not
    differentiable: a backward pass through the scales raises."""
    if _hip.tracked(x):
        return _hip.undifferentiated("quantize_rows", lambda: quantize_rows(x), x)
    x, ld = _rows(x, "quantize_rows")
    if x.dtype not in FLOATS:
        raise RuntimeError(f"quantize_rows: x must be float32, float16 or bfloat16, got {x.dtype}")
    rows, cols = x.shape
    q = torch.empty(rows, cols, dtype=torch.int8, device=x.device)
    scale = torch.empty(rows, dtype=torch.float32, device=x.device)
    _hip.call("fly_quantize_rows", x.device.index, x.data_ptr(), FLOATS[x.dtype], ld, rows, cols, q.data_ptr(),
              max(cols, 1), scale.data_ptr())
    return q, scale


class Int8Linear:
    """y = x W^T + b with W (channels, k) in 8 bits.  The weight is laid out for the matrix cores once, here; the object
    keeps no reference to the tensors: they are constants to autograd.  Calls run on the current stream with scratch from
    torch's allocator."""

    def __init__(self, weight: torch.Tensor, scale: torch.Tensor, bias: torch.Tensor | None = None):
        weight, ld = _rows(weight, "Int8Linear")
        self.n, self.k = weight.shape
        self.device = weight.device
        if weight.dtype != torch.int8:
            raise RuntimeError(f"Int8Linear: the weight must be int8, got {weight.dtype}")
        for name, t in (("scale", scale), ("bias", bias)):
            if t is not None and (t.dtype != torch.float32 or t.shape != (self.n,) or t.device != weight.device):
                raise RuntimeError(f"Int8Linear: {name} must be float32 of shape ({self.n},) on {weight.device}, "
                                   f"got {t.dtype} {tuple(t.shape)} on {t.device}")
        scale = scale.contiguous()
        bias = bias.contiguous() if bias is not None else None
        handle = ctypes.c_void_p()
        with torch.cuda.device(weight.device):
            _hip.check(_hip.load().fly_int8_create(weight.data_ptr(), ld, scale.data_ptr(), _hip.ptr(bias), self.n,
                                                   self.k, _hip.stream(weight.device), ctypes.byref(handle)),
                       "fly_int8_create")
        self._plan = _hip.Handle(handle, "fly_int8_destroy")

    @classmethod
    def from_float(cls, weight: torch.Tensor, bias: torch.Tensor | None = None) -> "Int8Linear":
        """A float weight, quantised with a scale for each channel."""
        q, scale = quantize_rows(weight.detach())
        return cls(q, scale, bias.detach().float() if bias is not None else None)

    def __call__(self, x: torch.Tensor, out_dtype: torch.dtype = torch.float32,
                 scale: torch.Tensor | None = None) -> torch.Tensor:
        """x (rows, k) float32, float16 or bfloat16; or int8 with the rows' scales.  Returns (rows, channels).  Not
        differentiable: a backward pass through the outputs raises."""
        if _hip.tracked(x) or (scale is not None and _hip.tracked(scale)):
            return _hip.undifferentiated("Int8Linear", lambda: self(x, out_dtype, scale), x, scale)
        x, ld = _rows(x, "Int8Linear")
        rows, k = x.shape
        dev = x.device
        if k != self.k or dev != self.device:
            raise RuntimeError(f"Int8Linear: x must be (rows, {self.k}) on {self.device}, got {tuple(x.shape)} on {dev}")
        x_type, y_type = _hip.TYPES.get(x.dtype), FLOATS.get(out_dtype)
        if x_type is None or y_type is None:
            raise RuntimeError(f"Int8Linear: x must be float32, float16, bfloat16 or int8 and out_dtype one of the "
                               f"floats, got {x.dtype} and {out_dtype}")
        if (x_type == 3) != (scale is not None):
            raise RuntimeError("Int8Linear: int8 rows come with their scales, other rows without")
        if scale is not None:
            if scale.dtype != torch.float32 or scale.shape != (rows,) or scale.device != dev:
                raise RuntimeError(f"Int8Linear: scale must be float32 of shape ({rows},) on {dev}, "
                                   f"got {scale.dtype} {tuple(scale.shape)} on {scale.device}")
            scale = scale.contiguous()
        y = torch.empty(rows, self.n, dtype=out_dtype, device=dev)
        handle = self._plan.handle
        need = _hip.load().fly_int8_workspace(handle, x_type, rows)
        ws = _hip.workspace(need, dev) if need else None
        _hip.call("fly_int8_linear", dev.index, handle, x.data_ptr(), x_type, ld, _hip.ptr(scale), rows, y.data_ptr(),
                  y_type, self.n, _hip.ptr(ws), need)
        return y
