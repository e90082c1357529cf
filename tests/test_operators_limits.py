"""CPU tests of the ends of what the 8-bit and distillation entry points accept: refused before any launch."""

from __future__ import annotations

import ctypes

import pytest

from test_operators_host import P, _distill, _refused, _top, lib  # noqa: F401


@pytest.mark.parametrize("call", [_top, _distill])
def test_temperatures_whose_scale_overflows(lib, call):  # noqa: F811
    """log2(e) / T is what the logits are multiplied with; 1 / T alone is still finite here."""
    for t in (2.95e-39, 3.5e-39, 4.2e-39):
        _refused(call(lib, temperature=t), lib, b"temperature")


@pytest.mark.parametrize("n,k", [(1 << 28, 1), ((1 << 28) + 1, 64), (1 << 23, 100_000), (1 << 22, (1 << 17) - 1), (1 << 27, 512)])
def test_weights_past_a_launch(lib, n, k):  # noqa: F811
    """Laying them out, or a product of one row, would take 2^32 threads, where a grid wraps without an error."""
    out = ctypes.c_void_p()
    _refused(lib.fly_int8_create(P, k, P, None, n, k, None, ctypes.byref(out)), lib, b"size")
