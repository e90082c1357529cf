"""CPU tests that pin the read-out loss's oracle: closed forms, and its gradients by differences."""

from __future__ import annotations

import numpy as np
import pytest

from oracle import readout as O


def test_closed_forms():
    x, w = np.zeros((3, 2)), np.zeros((4, 2))
    index = np.array([[1], [-1], [2]])
    loss, dx, dw, db = O.loss(x, w, None, index)
    assert np.allclose(loss, [np.log(4), 0, np.log(4)])
    assert np.allclose(db, np.array([.25, .25, .25, .25]) * 2 - np.array([0, 1, 1, 0]))
    legal = np.array([[1, 1, 0, 0], [1, 1, 1, 1], [0, 0, 0, 0]])
    loss, _, _, db = O.loss(x, w, None, index, legal=legal)
    assert np.allclose(loss, [np.log(2), 0, 0]) and np.allclose(db, [.5, -.5, 0, 0])
    assert np.isnan(O.loss(x, w, None, np.array([[4], [0], [0]]))[0][0])


@pytest.mark.parametrize("seed", range(4))
def test_gradients_by_differences(seed):
    g = np.random.default_rng(seed)
    rows, d, v, k = 5, 4, 7, 3
    x, w, b = g.normal(size=(rows, d)), g.normal(size=(v, d)), g.normal(size=v)
    index, weight = g.integers(-1, v, (rows, k)), g.normal(size=(rows, k))
    legal, scale = g.random((rows, v)) < 0.7, g.normal(size=rows)
    total = lambda: (O.loss(x, w, b, index, weight, legal)[0] * scale).sum()
    _, *grads = O.loss(x, w, b, index, weight, legal, scale)
    for t, got in zip((x, w, b), grads):
        for at in np.ndindex(t.shape):
            was, h = t[at], 1e-5
            t[at] = was + h
            up = total()
            t[at] = was - h
            down = total()
            t[at] = was
            assert abs((up - down) / (2 * h) - got[at]) < 1e-7


def test_clip():
    norm, (a,) = O.clip([np.array([3.0, 4.0])], 1.0)
    assert norm == 5 and np.allclose(a, np.array([3, 4]) / 5, rtol=1e-6)
    norm, (a, b) = O.clip([np.array([3.0]), np.array([-7.0, 1.0])], 14.0, np.inf)
    assert norm == 7 and a[0] == 3 and b[0] == -7
    assert O.clip([], 1.0) == (0.0, [])
