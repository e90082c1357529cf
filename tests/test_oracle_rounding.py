"""CPU tests of the oracle's bounds for each row: a plain float32 evaluation that takes differences before the scale keeps them,
one that scales first passes them where the logits are large, and a row's bound does not depend on the other rows."""

from __future__ import annotations

import numpy as np
import pytest

from oracle import operators as O


def _float32_loss(z, values, index, tail, temperature, scale_first=False):
    f = np.float32
    z, values, s = z.astype(f), values.astype(f), f(1) / f(temperature)
    out = np.zeros(len(z), f)
    for r in range(len(z)):
        rest = np.ones(z.shape[1], bool)
        rest[index[r]] = False
        parts = []
        for v in (z[r, rest], z[r, index[r]], values[r]):
            top = v.max()
            part = np.exp(v * s - f(top * s)) if scale_first else np.exp((v - top) * s)
            parts.append((top, part.sum(dtype=f)))
        (rt, rs), (lt, ls), (vt, vs) = parts
        m = max(rt, lt)
        ln_z = np.log(rs * np.exp((rt - m) * s) + ls * np.exp((lt - m) * s))
        x, at = vt * s, f(tail[r])
        ma = max(x, at)
        ln_a = np.log(vs * np.exp(x - ma) + np.exp(at - ma))
        logp = np.append((values[r] - vt) * s + (x - ma) - ln_a, at - ma - ln_a)
        logq = np.append((z[r, index[r]] - m) * s - ln_z, (rt - m) * s + np.log(rs) - ln_z)
        p, q = np.exp(logp), np.exp(logq)
        with np.errstate(invalid="ignore", over="ignore"):
            out[r] = f(temperature) ** 2 * np.where(p > 0, p * (logp - logq) - p + q, q).sum(dtype=f)
    return out


@pytest.mark.parametrize("shift", [0.0, -1e3, 3e4])
@pytest.mark.parametrize("temperature", [0.5, 1.0, 3.0])
def test_differences_first_keep_the_bound(shift, temperature):
    rng = np.random.default_rng(1)
    z = rng.normal(0, 3, (6, 500)).astype(np.float32) + np.float32(shift)
    t = rng.normal(0, 3, (6, 500)).astype(np.float32)
    values, index, tail = O.top(t, 20, temperature)
    tail = tail.astype(np.float32)
    loss, _, size, _ = O.distill(z, values, index, tail, temperature)
    off = O.row_rounding(z, values, tail, temperature)
    assert off.max() < 1e-4
    assert np.all(np.abs(_float32_loss(z, values, index, tail, temperature) - loss) <= 4 * off * size)


def test_scaling_first_passes_the_bound():
    rng = np.random.default_rng(1)
    z, t = (rng.normal(0, 3, (6, 500)).astype(np.float32) for _ in range(2))
    z += np.float32(3e6)
    values, index, tail = O.top(t, 20, 1.5)
    loss, _, size, _ = O.distill(z, values, index, tail, 1.5)
    off = O.row_rounding(z, values, tail, 1.5)
    wrong = _float32_loss(z, values, index, tail.astype(np.float32), 1.5, scale_first=True)
    assert not np.all(np.abs(wrong - loss) <= 4 * off * size)
    assert np.all(np.abs(_float32_loss(z, values, index, tail.astype(np.float32), 1.5) - loss) <= 4 * off * size)


def test_a_row_does_not_loosen_another():
    rng = np.random.default_rng(2)
    z = rng.normal(0, 3, (3, 100))
    values, index, tail = O.top(z, 5, 1.0)
    before = O.row_rounding(z, values, tail, 1.0), O.tail_rounding(z, index, 1.0)
    z[1] = -3.4e38
    z[2, ::2] = np.nan
    values2, index2, tail2 = O.top(z, 5, 1.0)
    after = O.row_rounding(z, values2, tail2, 1.0), O.tail_rounding(z, index2, 1.0)
    assert before[0][0] == after[0][0] and before[1][0] == after[1][0]
    assert after[0][0] < 1e-4 and after[1][0] < 1e-4
    # only what is visible counts
    legal = np.ones(z.shape, bool)
    legal[0, 7] = False
    z[0, 7] = 1e30
    assert O.row_rounding(z, values, tail, 1.0, legal)[0] <= before[0][0]


@pytest.mark.parametrize("shift", [-1e12, 1e20, -3.4e38])
def test_the_oracle_keeps_a_distribution_of_huge_logits(shift):
    """Equal logits are the uniform distribution wherever they lie: loss and gradient in closed form."""
    z, t = np.full((1, 20), shift), np.log(np.arange(1, 21))[None]
    values, index, tail = O.top(t, 3, 1.0)
    for t in (tail, None):
        loss, grad, _, _ = O.distill(z, values, index, t, 1.0)
        p = np.append(np.array([20.0, 19.0, 18.0]), 0.0 if t is None else 153.0)
        p /= p.sum()
        q = np.array([0.05, 0.05, 0.05, 0.85])
        on = p > 0
        assert loss[0] == pytest.approx(np.sum(p[on] * np.log(p[on] / q[on])))
        want = np.full(20, (q[3] - p[3]) / 17)
        want[index[0]] = q[:3] - p[:3]
        assert np.allclose(grad[0], want)
