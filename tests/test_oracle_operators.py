"""CPU tests of the operators' oracle: closed forms, and its gradient against differences of its loss."""

from __future__ import annotations

import numpy as np
import pytest

from oracle import operators as O


def test_quantise_by_hand():
    q, s = O.quantize(np.array([[0.0, 127.0, -63.5, 0.5, 1.5], [0, 0, 0, 0, 0], [1, np.nan, 0, 0, 0],
                                [1e-38, 0, 0, 0, 0]], np.float32))
    assert q[0].tolist() == [0, 127, -64, 0, 2] and s[0] == 1.0      # halves go to the even neighbour
    assert not q[1:].any() and s[1] == 0 and np.isnan(s[2]) and s[3] == 0


def test_top_by_hand():
    z = np.array([[1.0, 3.0, 3.0, -np.inf, 2.0, 3.0]])
    v, i, t = O.top(z, 2, 1.0)
    assert i.tolist() == [[1, 2]] and v.tolist() == [[3, 3]]
    assert t[0] == pytest.approx(np.log(np.exp(1) + np.exp(2) + np.exp(3)))
    v, i, t = O.top(z, 4, 1.0, legal=np.array([[1, 0, 1, 1, 0, 0]]))
    assert i.tolist() == [[2, 0, -1, -1]] and t[0] == -np.inf


def test_loss_is_the_divergence_when_everything_is_listed():
    rng = np.random.default_rng(0)
    z, t = rng.normal(0, 2, (3, 9)), rng.normal(0, 2, (3, 9))
    values, index, tail = O.top(t, 9, 2.0)
    loss, grad, _, _ = O.distill(z, values, index, tail, 2.0)
    p = np.exp(t / 2) / np.exp(t / 2).sum(1, keepdims=True)
    q = np.exp(z / 2) / np.exp(z / 2).sum(1, keepdims=True)
    assert np.allclose(loss, 4 * (p * np.log(p / q)).sum(1))
    assert np.allclose(grad, 2 * (q - p))


@pytest.mark.parametrize("k,with_tail,masked", [(3, True, False), (3, False, False), (5, True, True), (12, False, True)])
def test_gradient_against_differences(k, with_tail, masked):
    rng = np.random.default_rng(k)
    z, t = rng.normal(0, 2, (4, 11)), rng.normal(0, 2, (4, 11))
    legal = None
    if masked:
        legal = rng.random((4, 11)) < 0.6
        legal[1] = False
    values, index, tail = O.top(t, k, 1.5, legal)
    tail = tail if with_tail else None
    f = lambda x: O.distill(x, values, index, tail, 1.5, legal)[0]
    grad = O.distill(z, values, index, tail, 1.5, legal)[1]
    eps = 1e-6
    for j in range(11):
        e = np.zeros_like(z)
        e[:, j] = eps
        assert np.allclose((f(z + e) - f(z - e)) / (2 * eps), grad[:, j], atol=1e-7)
