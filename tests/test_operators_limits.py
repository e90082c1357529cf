"""CPU tests of the ends of what the 8-bit and distillation entry points accept: refused before any launch."""

from __future__ import annotations

import pytest

from test_operators_host import _distill, _refused, _top, lib  # noqa: F401


@pytest.mark.parametrize("call", [_top, _distill])
def test_temperatures_whose_scale_overflows(lib, call):  # noqa: F811
    """log2(e) / T is what the logits are multiplied with; 1 / T alone is still finite here."""
    for t in (2.95e-39, 3.5e-39, 4.2e-39):
        _refused(call(lib, temperature=t), lib, b"temperature")
