"""GPU tests of the read-out loss where one row says little of the others: rows and columns of zeros beside small ones, rows whose factor
is 0, batches in pieces.  Against the float64 oracle within its bounds, on the kernels of few rows and of many."""

from __future__ import annotations

import numpy as np
import numpy as np
import pytest
import torch

from oracle import readout as O
from test_gpu_readout import DEV, FEW, MANY, call, case, check, numpy, on

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


@pytest.mark.parametrize("rows", [FEW, MANY])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_rows_whose_factor_is_0_keep_what_they_hold(dtype, rows):
    """row_scale 0 takes a row's loss out of the sum: its NaN and infinities reach no gradient, its loss is what it is."""
    t = list(case(rows, 50, 60, dtype, k=3, legal=True))
    out = [8, 9, 13, rows - 1]
    t[3][out] = t[3][out].abs()
    t[5][out] = True
    scale = torch.ones(rows)
    scale[out] = 0.0
    want = call(*t, row_scale=scale.to(DEV))
    check(want, t, dtype, scale.double().numpy())
    x = t[0].clone()
    x[8], x[9, 3], x[13, 49], x[rows - 1] = float("nan"), float("inf"), -float("inf"), float("inf")
    loss, grads = call(x, *t[1:], row_scale=scale.to(DEV))
    kept = scale.to(DEV) != 0
    assert loss[~kept].isnan().all() and torch.equal(loss[kept], want[0][kept])
    assert not grads.x[~kept].any() and all(torch.equal(p, q) for p, q in zip(grads, want[1]))


@pytest.mark.parametrize("rows", [FEW, MANY])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_part_of_the_losses_taken_for_the_gradient(dtype, rows):
    """Selecting some rows' losses gives the others an upstream gradient of 0."""
    from chessfly.readout import Visits, readout_loss
    x, w, b, index, weight, _ = on(*case(rows, 50, 60, dtype, k=3))
    keep = torch.arange(rows, device=DEV) % 3 != 0
    bad = x.clone()
    bad[~keep] = float("inf")
    grads = []
    for rows_of_x in (x, bad):
        leaves = [p.clone().requires_grad_() for p in (rows_of_x, w, b)]
        readout_loss(*leaves, Visits(index, weight), reduction="none")[keep].mean().backward()
        grads.append([p.grad for p in leaves])
    assert all(p.isfinite().all() and torch.equal(p, q) for p, q in zip(*grads))


@pytest.mark.parametrize("rows", [FEW, MANY])
def test_all_factors_0(rows):
    t = case(rows, 50, 60, "float32", k=3)
    loss, grads = call(*t, grad_scale=0.0)
    assert loss.isfinite().all() and not any(g.any() for g in grads)


def _within(got, want, most):
    off = np.abs(got.double().cpu().numpy() - want)
    assert (off <= most).all(), float((off / most).max())


@pytest.mark.parametrize("rows", [FEW, MANY])
def test_large_rows_of_the_weight_that_no_row_sees(rows):
    """The others, 2^20 times smaller, are within the bounds of a weight without any large row."""
    x, w, b, index, weight, legal = case(rows, 64, 90, "float32", seed=rows, k=3, legal=True)
    hidden = torch.arange(90) % 6 == 1
    legal = legal & ~hidden
    small = w * 2.0 ** -20
    w = torch.where(hidden[:, None], w, small)
    loss, grads = call(x, w, b, index, weight, legal)
    args = numpy(x, w, b, index, weight, legal)
    n = lambda m: (m[0], m[1], m[2], m[3], "float32", *m[4:])
    want, most = O.loss(*args), O.bounds(*n(numpy(x, small, b, index, weight, legal)))
    for got, e, m in zip((loss, *grads), want, most):
        _within(got, e, m)


@pytest.mark.parametrize("rows", [2 * FEW, MANY])
def test_large_rows_of_x_that_see_other_columns(rows):
    """What rows 2^20 times smaller give their columns is within the bounds of those rows alone."""
    x, w, b, index, weight, _ = case(rows, 64, 90, "float32", seed=rows, k=3)
    half = rows // 2
    legal = torch.zeros(rows, 90, dtype=torch.bool)
    legal[:half, :45] = legal[half:, 45:] = True
    index = index % 45
    index[half:] += 45
    x[half:] *= 2.0 ** -20
    loss, grads = call(x, w, b, index, weight, legal)
    part = numpy(*(t[half:] if t.shape[0] == rows else t for t in (x, w, b, index, weight, legal)))
    want, most = O.loss(*part), O.bounds(*part[:4], "float32", *part[4:])
    _within(loss[half:], want[0], most[0])
    _within(grads.x[half:], want[1], most[1])
    _within(grads.weight[45:], want[2][45:], most[2][45:])
    _within(grads.bias[45:], want[3][45:], most[3][45:])


@pytest.mark.parametrize("of", ["x", "weight"])
@pytest.mark.parametrize("size", [1e-20, 1e-28, 1e-30, 1e-32, 1e-34])
@pytest.mark.parametrize("rows", [FEW, MANY])
def test_small_rows_and_the_mean_over_them(rows, size, of):
    """The largest of the gradients about size / rows: far above float32's smallest number, as the factors on the way there need not be."""
    t = list(case(rows, 64, 90, "float32", seed=rows, k=3))
    t[of == "weight"] = t[of == "weight"] * size
    check(call(*t, grad_scale=1 / rows), t, "float32", np.full(rows, 1 / rows))
