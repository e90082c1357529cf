"""Oracle: the 8-bit dense map and distillation from a teacher's top logits, in float64 numpy, row by row.
TEST INFRASTRUCTURE ONLY (imported by tests/; never by the product).  No counterpart in the reference.

  quantize     rows to 8 bits in the float32 arithmetic that defines the operator: q, scale
  int8_linear  (sum q w) (s t) + b, and the bound of a float32 evaluation of it
  top          the k largest visible logits, ties to the lower column, and the rest's log-sum-exp
  distill      loss and gradient by the formulas, row by row
  rounding     what a float32 evaluation of top and distill may be off in an exponent, by the largest logit of all rows
  row_rounding, tail_rounding   the same for each row by its own logits, where differences are taken before the scale
"""

from __future__ import annotations

import numpy as np

UNIT = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}   # half a unit in the last place, relative
TINY = {"float32": 2.0 ** -149, "float16": 2.0 ** -25, "bfloat16": 2.0 ** -134}  # and below the normal numbers


def quantize(x: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    x = np.asarray(x, dtype=np.float32)
    q = np.zeros(x.shape, np.int8)
    scale = np.zeros(x.shape[0], np.float32)
    for r, row in enumerate(x):
        if not np.all(np.isfinite(row)):
            scale[r] = np.nan
            continue
        top = np.float32(np.abs(row).max()) if row.size else np.float32(0)
        if top < np.float32(2.0 ** -120):
            continue
        scale[r] = top / np.float32(127)
        q[r] = np.rint(row * (np.float32(127) / top)).astype(np.int8)
    return q, scale


def int8_linear(q, s, w, t, b):
    """y in float64 and the bound: the sum's, the scales', their product's and the bias's roundings to float32."""
    acc = q.astype(np.float64) @ w.astype(np.float64).T
    part = acc * (s.astype(np.float64)[:, None] * t.astype(np.float64)[None, :])
    bias = np.zeros(w.shape[0]) if b is None else b.astype(np.float64)
    return part + bias, 4 * 2.0 ** -24 * (np.abs(part) + np.abs(bias))


def _lse(v: np.ndarray) -> float:
    if v.size == 0 or v.max() == -np.inf:
        return -np.inf
    m = v.max()
    return float(m + np.log(np.exp(v - m).sum()))


def _parts(v: np.ndarray, temperature: float) -> tuple[float, float]:
    """The largest of v (0 where there is none but -inf), and log sum exp((v - it) / temperature)."""
    if v.size == 0 or v.max() == -np.inf:
        return 0.0, -np.inf
    m = v.max()
    return float(m), float(np.log(np.exp((v - m) / temperature).sum()))


def top(z: np.ndarray, k: int, temperature: float, legal=None):
    rows, cols = z.shape
    z = np.asarray(z, dtype=np.float64)
    values = np.full((rows, k), -np.inf)
    index = np.full((rows, k), -1, np.int32)
    tail = np.full(rows, -np.inf)
    for r in range(rows):
        seen = z[r] != -np.inf
        if legal is not None:
            seen &= legal[r] != 0
        cand = np.nonzero(seen)[0]
        key = np.where(np.isnan(z[r, cand]), np.inf, z[r, cand])
        # NaN above all numbers, +inf included
        order = np.lexsort((cand, -key, ~np.isnan(z[r, cand])))
        cand = cand[order]
        n = min(k, len(cand))
        values[r, :n] = z[r, cand[:n]]
        index[r, :n] = cand[:n]
        tail[r] = _lse(z[r, cand[n:]] / temperature)
    return values, index, tail


def distill(z, values, index, tail, temperature: float, legal=None):
    """loss (rows), dloss/dz (rows, cols), and of each the size that its rounding error is proportional to: sum p |log(p/q)|
    plus 1, and the two terms of each gradient added instead of subtracted."""
    z = np.asarray(z, dtype=np.float64)
    rows, cols = z.shape
    loss, size = np.zeros(rows), np.zeros(rows)
    grad, parts = np.zeros((rows, cols)), np.zeros((rows, cols))
    T = float(temperature)
    for r in range(rows):
        idx = index[r]
        listed = [i for i in range(len(idx)) if idx[i] >= 0 and (idx[i] >= cols or legal is None or legal[r, idx[i]])]
        cols_of = [int(idx[i]) for i in listed]
        if any(c >= cols for c in cols_of) or len(set(cols_of)) < len(cols_of):
            loss[r], grad[r] = np.nan, np.nan
            continue
        # differences come before the scale: a float64 has no digits left for a logarithm next to logits of 1e12
        zr = z[r] if legal is None else np.where(legal[r] != 0, z[r], -np.inf)
        rest = np.ones(cols, bool)
        rest[cols_of] = False
        rest_top, rest_log = _parts(zr[rest], T)
        has_rest = rest_log != -np.inf
        at = -np.inf if tail is None or not has_rest else float(tail[r])
        v = np.asarray(values[r], np.float64)[listed]
        if (v.size == 0 or v.max() == -np.inf) and at == -np.inf or np.all(zr == -np.inf):
            continue
        m = zr.max()
        ln_z = _parts(zr, T)[1]
        logq = np.append((zr[cols_of] - m) / T - ln_z, (rest_top - m) / T + rest_log - ln_z if has_rest else -np.inf)
        v_top, v_log = _parts(v, T)
        x = v_top / T if v_log != -np.inf else -np.inf
        ma = max(x, at)
        ln_a = np.log(np.exp(x - ma + v_log) + np.exp(at - ma))
        logp = np.append((v - v_top) / T + (x - ma) - ln_a, at - ma - ln_a)
        p, q = np.exp(logp), np.exp(logq)
        with np.errstate(invalid="ignore"):
            d = np.where(p > 0, logp - logq, 0.0)
        loss[r] = T * T * float(np.sum(np.where(p > 0, p * d, 0.0)))
        size[r] = T * T * (1.0 + float(np.sum(np.where(p > 0, p * np.abs(d), 0.0))))
        if has_rest:
            share = np.exp((zr - rest_top) / T - rest_log)
            grad[r] = np.where(rest, T * share * (q[-1] - p[-1]), 0.0)
            parts[r] = np.where(rest, T * share * (q[-1] + p[-1]), 0.0)
        grad[r, cols_of] = T * (q[:-1] - p[:-1])
        parts[r, cols_of] = T * (q[:-1] + p[:-1])
    return loss, grad, size, parts


def rounding(z, values, temperature: float, threads: int = 64) -> float:
    """How far an exponent z / T - (a log-sum-exp) may be off in float32: the scaled logit's two roundings, the difference's
    and the log-sum-exp's own, each 2^-24 of the largest scaled logit; the exponential and the logarithm (2 units each);
    and the sum, a thread's share of the columns one after the other, then a tree."""
    big = 0.0
    for v in (z, values):
        v = np.asarray(v, dtype=np.float64)
        v = v[np.isfinite(v)]
        big = max(big, float(np.abs(v).max()) / temperature if v.size else 0.0)
    terms = -(-np.asarray(z).shape[1] // threads)
    return (6 * big + terms + 24) * 2.0 ** -24


MOST = 110.0        # exp of less than -MOST is 0 in float32: a difference past it adds no error
LEAST = 2.0 ** -124  # four of float32's smallest normal numbers, below which an exponential may count as 0


def _spread(v: np.ndarray, temperature: float) -> float:
    v = np.asarray(v, dtype=np.float64)
    v = v[np.isfinite(v)]
    return min(float(v.max() - v.min()) / temperature, MOST) if v.size else 0.0


def _terms(z, threads: int) -> int:
    return -(-np.asarray(z).shape[1] // threads) + 24


def row_rounding(z, values, tail, temperature: float, legal=None, threads: int = 64) -> np.ndarray:
    """How far an exponent of distill may be off in each row.  Differences of logits come before the scale, so a row's error
    does not depend on where its logits lie but on how far they spread: 2^-24 of a difference / T for it, the scale (its two
    roundings) and the product, through up to three maxima (a thread's, a list's or the rest's, the row's), whose steps add
    up to no more than the spread: 6 spreads, of the student and of the list.  The teacher's tail is scaled already: where it
    is near the list's largest entry, that one is scaled too, two roundings of its size.  The sum and the functions as in
    `rounding`."""
    off = np.zeros(len(z))
    for r in range(len(z)):
        seen = z[r] if legal is None else np.asarray(z[r])[np.asarray(legal[r]) != 0]
        size = 6 * (_spread(seen, temperature) + _spread(values[r], temperature))
        v = np.asarray(values[r], np.float64)
        v = v[np.isfinite(v)]
        if tail is not None and np.isfinite(tail[r]) and v.size and abs(v.max() / temperature - tail[r]) < MOST + 10:
            size += 2 * abs(v.max()) / temperature
        off[r] = size
    return (off + _terms(z, threads)) * 2.0 ** -24


def tail_rounding(z, index, temperature: float, legal=None, threads: int = 64) -> np.ndarray:
    """How far the tail of top may be off in each row: the spread of what is not listed, taken from a bound that lies at most
    MOST / 2 above it, as above; and four roundings of its largest logit / T (the bound's scaling, 1 / T, its product, the
    sum)."""
    off = np.zeros(len(z))
    for r in range(len(z)):
        rest = np.ones(len(z[r]), bool) if legal is None else np.asarray(legal[r]) != 0
        rest[[c for c in index[r] if c >= 0]] = False
        v = np.asarray(z[r], np.float64)[rest]
        v = v[np.isfinite(v)]
        off[r] = 6 * (_spread(v, temperature) + MOST / 2) + 4 * (abs(v.max()) / temperature if v.size else 0.0)
    return (off + _terms(z, threads)) * 2.0 ** -24
