"""GPU tests at the ends of what the 8-bit and distillation entry points accept."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
ROWS = (1 << 26) + 5        # 64 threads for each row are 2^32, more than a launch holds
PARTS = [(i, min(i + (1 << 24) + 3, ROWS)) for i in range(0, ROWS, (1 << 24) + 3)]


def _rows(cols, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(ROWS, cols, generator=g, device=DEV, dtype=torch.float16)


def test_more_rows_than_a_launch_holds_to_8_bits():
    from chessfly.int8 import quantize_rows
    x = _rows(1, 1)
    whole = quantize_rows(x)
    for a, b in PARTS:
        assert all(torch.equal(w[a:b], p) for w, p in zip(whole, quantize_rows(x[a:b])))


def test_more_rows_than_a_launch_holds_of_logits():
    from chessfly.distill import TopLogits, distill_loss_and_grad, top_logits
    z = _rows(2, 1)
    legal = torch.rand(ROWS, 2, device=DEV) < 0.9
    lists = top_logits(_rows(2, 2), 1, 2.0, legal)
    scale = torch.rand(ROWS, device=DEV)
    whole = distill_loss_and_grad(z, lists, 2.0, legal, row_scale=scale)
    for a, b in PARTS:
        assert all(torch.equal(w[a:b], p) for w, p in zip(lists, top_logits(_rows(2, 2)[a:b], 1, 2.0, legal[a:b])))
        part = distill_loss_and_grad(z[a:b], TopLogits(*(t[a:b] for t in lists)), 2.0, legal[a:b], row_scale=scale[a:b])
        assert all(torch.equal(w[a:b], p) for w, p in zip(whole, part))
