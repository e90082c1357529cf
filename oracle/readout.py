"""Oracle: a read-out's softmax cross entropy with its gradients, and clipping by the gradients' norm, in float64 numpy.
TEST INFRASTRUCTURE ONLY (imported by tests/; never by the product).  No counterpart in the reference.

  loss      rows' losses and the gradients by x, w and b, from the formulas, row by row over the list of targets
  bounds    how far a float32 evaluation of them may be off, element by element, by the roundings that it makes
  clip      the norm and the scaled gradients
"""

from __future__ import annotations

import numpy as np

from .operators import TINY, UNIT

U = 2.0 ** -24
# The operands' own roundings: 16-bit floats are multiplied exactly; float32 ones as two halves, 2^-22 of the value each (a half
# of a half's residual), the product of the two low parts left out another 2^-22.
OPERAND = {"float32": 3 * 2.0 ** -22, "float16": 0.0, "bfloat16": 0.0}
# u as it is multiplied: one rounding to the 16-bit type, or two halves; float16 holds 2^14 u down to 2^-24 steps, the low half 2^11 finer.
HELD = {"float32": 2.0 ** -22, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
# With 16-bit operands the logits wait for their rows' sums as their distance from their part's largest, in 65,535 steps up to 32 and
# as none from there on: p errs by e^(half a step) - 1, or by e^-32 of the part's largest.
STEP = 16.0 / 65535 * (1 + 2.0 ** -11)
HELD_LEAST = {"float32": 2.0 ** -49, "float16": 2.0 ** -38, "bfloat16": 2.0 ** -120}


def _targets(index, weight, legal, rows, v):
    """Each row's summed weights by column (rows, v), sums of weights and of their sizes, and whether an index lies past v."""
    index = index.reshape(rows, -1)
    weight = np.ones(index.shape) if weight is None else weight.astype(np.float64)
    t, a, whole, bad = np.zeros((rows, v)), np.zeros(rows), np.zeros(rows), np.zeros(rows, bool)
    for r in range(rows):
        for c, x in zip(index[r], weight[r]):
            if c < 0 or x == 0:
                continue
            if c >= v:
                bad[r] = True
                continue
            if legal is not None and not legal[r, c]:
                continue
            t[r, c] += x
            a[r] += x
            whole[r] += abs(x)
    return t, a, whole, bad


def loss(x, w, b, index, weight=None, legal=None, scale=None):
    """loss (rows), dx, dw, db of sum(scale * loss); NaN rows where an index lies past the columns."""
    x, w = x.astype(np.float64), w.astype(np.float64)
    rows, v = x.shape[0], w.shape[0]
    z = x @ w.T + (0.0 if b is None else b.astype(np.float64))
    if legal is not None:
        z = np.where(legal.astype(bool), z, -np.inf)
    t, a, whole, bad = _targets(index, weight, legal, rows, v)
    some = whole != 0
    top = z.max(1, keepdims=True, initial=-np.inf)
    top = np.where(np.isfinite(top), top, 0.0)
    e = np.exp(z - top)
    total = e.sum(1, keepdims=True)
    with np.errstate(divide="ignore", invalid="ignore"):
        far = top + np.log(total) - z
        out = np.where(some, np.where(t != 0, t * far, 0.0).sum(1), 0.0)
        p = np.where(total > 0, e / total, 0.0)
    g = np.where(some[:, None], a[:, None] * p - t, 0.0)
    out[bad] = np.nan
    g[bad] = np.nan
    g *= (np.ones(rows) if scale is None else scale.astype(np.float64))[:, None]
    return out, g @ w, g.T @ x, g.sum(0)


def bounds(x, w, b, index, dtype, weight=None, legal=None, scale=None, bias_dtype=None):
    """Bounds of the four outputs' errors, for finite rows."""
    x, w = x.astype(np.float64), w.astype(np.float64)
    rows, d = x.shape
    v = w.shape[0]
    bias = np.zeros(v) if b is None else b.astype(np.float64)
    ax, aw = np.abs(x), np.abs(w)
    z = x @ w.T + bias
    # a logit: the operands, d sums in any order, scales and bias
    ez = (OPERAND[dtype] + (d + 40) * U) * (ax @ aw.T) + 4 * U * (np.abs(z) + np.abs(bias))
    seen = np.ones((rows, v), bool) if legal is None else legal.astype(bool)
    ez_row = np.where(seen, ez, 0.0).max(1)
    top = np.where(seen, z, -np.inf).max(1, initial=-np.inf)
    top = np.where(np.isfinite(top), top, 0.0)
    gap = np.where(seen, top[:, None] - z, 0.0)
    # log sum exp: the logits, the exponents' two products and the exponentials (2^-22), v sums in a tree of 64 lanes, the logarithm
    tree = (80 + v / 64) * U
    near = np.minimum(gap, 30.0).max(1)          # terms further down add less than their share of an error
    e_lse = ez_row + 3 * U * near + 2.0 ** -22 + tree + 2.0 ** -21 * np.log2(v + 2.0)
    t, a, whole, _ = _targets(index, weight, legal, rows, v)
    # n weights in any order err by (n - 1) U of their sizes' sum, which weights of both signs leave larger than their sum
    sizes = t if weight is None else _targets(index, np.abs(weight), legal, rows, v)[0]
    n = max(1, np.prod(index.shape) // max(rows, 1))
    lse_gap = np.where(seen, gap, 0.0) + np.log(v)
    e_loss = (np.abs(t) * (ez + e_lse[:, None] + 4 * U * lse_gap) + sizes * (n + 8) * U * (lse_gap + 1)).sum(1) \
        + whole * (e_lse + 1e-7)
    # u: p by its exponent, the weights' sums, and how it is held
    s = np.abs(np.ones(rows) if scale is None else scale.astype(np.float64))
    p = np.where(seen, np.exp(np.minimum(z - top[:, None], 0.0)), 0.0)
    p /= np.maximum(p.sum(1, keepdims=True), 1e-300)
    ep = p * np.expm1(ez + e_lse[:, None] + 6 * U * (gap + 1) + 2.0 ** -21)
    if dtype != "float32":
        listed = t != 0                      # the targets' own logits are kept in float32
        ep = ep + np.where(listed, 0.0, p * STEP * 1.01 + np.exp(-32.0))
    u_size = np.abs(a[:, None] * p - t)
    eg = np.abs(a)[:, None] * ep + (n + 8) * U * (whole[:, None] * p + sizes)
    held = HELD[dtype] * (u_size + eg) + 4 * U * u_size + 1e-38
    eg_row = (eg + held + HELD_LEAST[dtype] * whole[:, None]) * s[:, None]
    size = u_size * s[:, None]
    # a column's products take the rows' factors by the largest of them
    most = (whole * s * (ax.max(1) if dtype == "float32" else 1.0))
    weigh = np.divide(most.max(initial=0.0), ax.max(1) if dtype == "float32" else 1.0, out=np.zeros(rows),
                      where=(ax.max(1) > 0) if dtype == "float32" else np.ones(rows, bool))
    eg_col = (eg + held) * s[:, None] + HELD_LEAST[dtype] * 4 * weigh[:, None]
    # and a row's the weights' units: the largest row's against each
    if dtype == "float32":
        wide = aw.max(1)
        eg_row = eg_row + HELD_LEAST[dtype] * 4 * (whole * s)[:, None] * np.divide(wide.max(), wide, out=np.zeros(v), where=wide > 0)[None]
    op = OPERAND[dtype]
    dx = eg_row @ aw + (op + (v + 40) * U) * ((size + eg_row) @ aw)
    dw = eg_col.T @ ax + (op + (rows + 40) * U) * ((size + eg_col).T @ ax)
    db = (eg * s[:, None]).sum(0) + (rows + 8) * U * size.sum(0)
    _, gx, gw, gb = loss(x, w, b, index, weight, legal, scale)
    bt = bias_dtype or dtype
    r = lambda e, g, ty: 1.01 * e + UNIT[ty] * 1.01 * np.abs(np.nan_to_num(g)) + TINY[ty]
    return 1.01 * e_loss + 1e-30, r(dx, gx, dtype), r(dw, gw, dtype), r(db, gb, bt)


def clip(grads, limit, norm_type=2.0):
    """The norm in float64, and the gradients scaled by limit / (norm + 1e-6) where that is below 1."""
    flat = [g.astype(np.float64).ravel() for g in grads]
    if norm_type == np.inf:
        norm = max([np.abs(f).max(initial=0.0) for f in flat], default=0.0)
    else:
        norm = float(np.sqrt(sum((f * f).sum() for f in flat)))
    scale = min(1.0, limit / (norm + 1e-6))
    return norm, [g.astype(np.float64) * scale for g in grads]
