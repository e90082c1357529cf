"""GPU tests of the read-out loss where one row says little of the others: rows and columns of zeros beside small ones, rows whose factor
is 0, batches in pieces.  Against the float64 oracle within its bounds, on the kernels of few rows and of many."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from test_gpu_readout import DEV, FEW, MANY, call, case, check, on

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("size", [1e-3, 1e-6, 1e-8, 1e-20, 1e-30])
@pytest.mark.parametrize("rows", [FEW, MANY])
def test_zero_rows_of_the_weight_take_no_bits_of_the_others(rows, size):
    """Moves never legal so far, padding of a vocabulary: among small rows, some of them targets."""
    x, w, b, index, weight, legal = case(rows, 64, 90, "float32", seed=rows, k=3)
    w = w * size
    w[[0, 17, 89]] = 0.0
    index[5] = 17
    t = (x, w, b, index, weight, legal)
    check(call(*t), t, "float32")


@pytest.mark.parametrize("size", [1e-3, 1e-6, 1e-8, 1e-20, 1e-30])
@pytest.mark.parametrize("rows", [FEW, MANY])
def test_zero_rows_of_x_take_no_bits_of_the_others(rows, size):
    """Positions without activity that have targets all the same, one of them of a large weight."""
    x, w, b, index, weight, legal = case(rows, 64, 90, "float32", seed=rows, k=3)
    index = index.abs()
    x = x * size
    x[[0, 21, rows - 1]] = 0.0
    weight[21] = 100.0
    t = (x, w, b, index, weight, legal)
    check(call(*t), t, "float32")


@pytest.mark.parametrize("rows", [FEW, MANY])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_nothing_but_zeros(dtype, rows):
    """A network's first step, whose read-out starts at zero, and a batch without activity."""
    x, w, b, index, weight, legal = case(rows, 40, 70, dtype, seed=3, k=3, legal=True)
    for t in ((x, torch.zeros_like(w), b, index, weight, legal), (torch.zeros_like(x), w, b, index, weight, legal)):
        loss, grads = got = call(*t)
        check(got, t, dtype)
        assert not (grads.x if not t[1].any() else grads.weight).any()
