"""GPU tests of top logits and distillation where the logits' values are out of the ordinary, each row within its own bound:
an extreme value in one row loosens no other (see oracle.operators.row_rounding and tail_rounding).

Tolerances, of an exponent that is off by e: the loss moves by its size (sum p |log(p/q)| + 1) times two of them (p's and q's),
doubled for the divergence's own terms; a gradient by its two parts times as much, plus its rounding to the logits' type.  What
is below the smallest normal float32 may count as 0."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import operators as O
from test_gpu_distill import DEV, FLOATS, INF, NAMES, _dev, _logits, _mask, _near, _np, _teacher

pytestmark = pytest.mark.gpu


def _check_top(z, k, temperature=1.0, legal=None):
    from chessfly.distill import top_logits
    got = top_logits(_dev(z), k, temperature, _dev(legal))
    with np.errstate(invalid="ignore"):
        values, index, tail = O.top(_np(z), k, temperature, _np(legal))
    assert np.array_equal(got.index.cpu().numpy(), index)
    assert np.array_equal(got.values.double().cpu().numpy(), values, equal_nan=True)
    _near(got.tail, tail, O.tail_rounding(_np(z), index, temperature, _np(legal)))


def _check_distill(z, teacher, temperature=1.0, legal=None):
    """The one-pass call, the loss alone, and autograd with a factor of its own for each row.  Returns the gradient."""
    from chessfly.distill import TopLogits, distill_loss, distill_loss_and_grad
    td, zd = TopLogits(*map(_dev, teacher)), _dev(z)
    kw = dict(temperature=temperature, legal=_dev(legal))
    loss, grad = distill_loss_and_grad(zd, td, **kw)
    with np.errstate(invalid="ignore", over="ignore"):
        ref, ref_grad, size, parts = O.distill(_np(z), *map(_np, teacher), temperature, _np(legal))
    off = O.row_rounding(_np(z), _np(teacher[0]), _np(teacher[2]), temperature, _np(legal))
    unit, tiny = O.UNIT[NAMES[z.dtype]], O.TINY[NAMES[z.dtype]]

    def check_grad(got, w):
        want = ref_grad * w
        tol = ((4 * off[:, None] + 8 * 2.0 ** -24) * np.abs(parts * w) + 1.01 * unit * np.abs(want) + tiny
               + O.LEAST * temperature * np.abs(w))
        past = np.isfinite(want) & (np.abs(want) + tol > torch.finfo(z.dtype).max)     # may round to an infinity
        assert not bool(torch.isnan(got)[torch.from_numpy(past).to(DEV)].any())
        _near(torch.where(torch.from_numpy(past).to(DEV), 0.0, got.double()), np.where(past, 0.0, want), tol)

    _near(loss, ref, 4 * off * size)
    check_grad(grad, np.ones((len(z), 1)))
    alone = distill_loss(zd, td, reduction="none", **kw)
    assert torch.equal(torch.nan_to_num(alone, 7.0), torch.nan_to_num(loss, 7.0))
    leaf = zd.detach().clone().requires_grad_(True)
    up = torch.linspace(0.25, 2.0, len(z))
    distill_loss(leaf, td, reduction="none", **kw).backward(_dev(up))
    check_grad(leaf.grad, _np(up)[:, None])
    return grad


# the fills that a program puts on moves that are not legal, and how far its logits spread with them
FILLS = [(torch.float32, f) for f in (-1e5, -1e9, -1e10, -1e12, -1e20, -1e30, -1e32, -3.4028234663852886e38)]
FILLS += [(torch.bfloat16, f) for f in (-1e9, -1e10, -1e12, -1e20, -1e30, -1e32, -3.3895313892515355e38)]
FILLS += [(torch.float16, f) for f in (-3e4, -65504.0)]


@pytest.mark.parametrize("cols", [300, 4168, 16390, 33000, 70000])
@pytest.mark.parametrize("dtype,fill", FILLS)
def test_illegal_moves_filled_with_a_large_negative_number(cols, dtype, fill):
    """No mask: the fill takes its place.  The list holds some of the 30 legal moves, all of them, and fills too."""
    g = torch.Generator().manual_seed(cols)
    z, t = _logits(5, cols, 1), _logits(5, cols, 2)
    for row in (0, 1, 2):
        hidden = torch.ones(cols, dtype=torch.bool)
        hidden[torch.randperm(cols, generator=g)[:30]] = False
        z[row, hidden] = t[row, hidden] = fill
    z[1] = fill                                             # nothing but fills
    z[3] = (z[3] * abs(fill) / 64).clamp(fill / 8, -fill / 8)   # logits of that size themselves
    z, t = z.to(dtype), t.to(dtype).float()
    f = lambda a: torch.from_numpy(a.astype(np.float32))
    for k, temperature in ((8, 1.0), (30, 1.0), (40, 1.0)) + (((8, 2.0), (30, 2.0)) if fill > -1e35 else ()):
        values, index, tail = O.top(_np(t), k, temperature)
        teacher = f(values), torch.from_numpy(index), f(tail)
        _check_distill(z, teacher, temperature)
        _check_distill(z, (*teacher[:2], None), temperature)
        _check_top(z, k, temperature)


@pytest.mark.parametrize("temperature", [1e-3, 1e-6])
def test_a_small_temperature_is_a_large_logit(temperature):
    for dtype in FLOATS:
        z = _logits(4, 4168, 3, dtype)
        _check_distill(z, _teacher(4, 4168, 8, 5, temperature, tail=False), temperature)
        _check_top(z, 8, temperature)


# register rows of 1, 2, 4 and 8 pieces a thread, and rows past them
@pytest.mark.parametrize("rows,cols", [(4, 300), (4, 4168), (4, 9000), (4, 20000), (4, 33000), (2, 70000), (1030, 1200)])
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("shift,temperature", [(-100.0, 1.0), (-1000.0, 1.0), (0.0, 0.02), (-60.0, 0.5), (1000.0, 1.0)])
def test_threads_that_see_nothing_of_a_row_that_lies_low(rows, cols, dtype, shift, temperature):
    """About 30 visible moves: most threads hold none.  The softmax does not see a constant added to all logits."""
    z = (_logits(rows, cols, 1) - 10 * (shift == 0) + shift).to(dtype)
    legal = _mask(rows, cols, 7, 30 / cols)
    legal[rows - 1, :20] = True
    hidden = torch.where(legal, z, torch.tensor(-INF, dtype=dtype))     # the same without a mask
    for k in (8, 64):
        teacher = _teacher(rows, cols, k, 5, temperature, legal)
        grad = _check_distill(z, teacher, temperature, legal)
        assert bool((grad[~legal.to(DEV)] == 0).all())
        assert torch.equal(_check_distill(hidden, teacher, temperature), grad)


@pytest.mark.parametrize("temperature", [1e-20, 1e-36, 1e20])
def test_temperatures_whose_square_leaves_the_range(temperature):
    for dtype in FLOATS:
        z = _logits(4, 4168, 3, dtype)
        _check_distill(z, _teacher(4, 4168, 8, 5, temperature, tail=temperature > 1), temperature)
        _check_top(z, 8, temperature)


def test_a_teacher_whose_scaled_logits_leave_the_range():
    z, (values, index, _) = _logits(4, 4168, 3, scale=0.3), _teacher(4, 4168, 8, 5, 1.0)
    _check_distill(z, (values / 10 + 10, index, None), 2e-38)


LENGTHS = [37, 300, 4168, 16390, 33000, 70000]


@pytest.mark.parametrize("cols", LENGTHS)
@pytest.mark.parametrize("dtype", FLOATS)
def test_top_of_odd_values_row_by_row(cols, dtype):
    low = torch.finfo(dtype).min
    z = _logits(10, cols, 3, dtype)
    z[0] = -INF
    z[1] = low
    z[2, ::3] = low
    z[3, ::2] = -INF
    z[4, 5] = INF
    z[5, [2, 9]] = float("nan")
    z[6] = -INF
    z[6, 11] = 2.0
    z[7] = torch.finfo(dtype).tiny
    z[7, 3] = -torch.finfo(dtype).tiny
    z[8] = -low
    z[9, 1::2] -= 1000
    for k, legal in ((1, None), (4, None), (30, _mask(10, cols, 4, 0.5)), (256, None)):
        _check_top(z, k, 1.0, legal)
        _check_top(z, k, 3.0, legal)


@pytest.mark.parametrize("cols", LENGTHS)
@pytest.mark.parametrize("dtype", FLOATS)
def test_distill_odd_values_row_by_row(cols, dtype):
    low = torch.finfo(dtype).min
    values, index, tail = _teacher(16, cols, 6, 3, 1.0)
    z = _logits(16, cols, 4, dtype)
    z[0] = -INF                                  # the student sees nothing
    z[1] = low
    z[2, ::3] = low
    z[3] = -INF
    z[3, index[3, 0].item()] = 1.0               # nothing but one listed move
    z[4, index[4, 1].item()] = -INF              # the teacher's move is impossible: infinite loss, finite gradient
    z[5, (index[5, 0].item() + 1) % cols] = float("nan")
    index[6] = -1                                # nothing listed: the tail alone
    index[7, 1:] = -1
    index[8, 0], index[8, 2] = -1, -5
    values[9, 3:] = -INF                         # listed, of no probability
    tail[10] = -INF
    z[11] += 40.0
    z[12], z[13] = -low, 0.0
    values[14] = torch.finfo(torch.float32).min  # the teacher lists what it masks
    values[15, 2:] = torch.finfo(torch.float32).min
    _check_distill(z, (values, index, tail))
    _check_distill(z, (values, index, None), 2.0)
    _check_distill(z, (values, index, tail), 1.0, _mask(16, cols, 3, 0.5))


def test_each_row_is_scaled_by_its_own_upstream_gradient():
    """Bit for bit the gradient that a factor for each row gives, and not the first row's factor."""
    from chessfly.distill import TopLogits, distill_loss, distill_loss_and_grad
    z, up = _logits(9, 700, 3).to(DEV), torch.linspace(-1.5, 2.0, 9).to(DEV)
    teacher = TopLogits(*map(_dev, _teacher(9, 700, 12, 5, 1.0)))
    leaf = z.clone().requires_grad_(True)
    distill_loss(leaf, teacher, reduction="none").backward(up)
    assert torch.equal(leaf.grad, distill_loss_and_grad(z, teacher, row_scale=up)[1])
    one = torch.zeros(9, device=DEV)
    one[4] = 1.0
    leaf.grad = None
    distill_loss(leaf, teacher, reduction="none").backward(one)
    assert bool((leaf.grad[torch.arange(9, device=DEV) != 4] == 0).all()) and bool((leaf.grad[4] != 0).any())
