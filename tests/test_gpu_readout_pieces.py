"""GPU tests of the read-out loss over more rows than a piece holds: lists, masks and factors of later pieces, what is kept of the first
one, gradients of the weight and bias over all of them.  Losses and dx have the bits of calls on each piece's rows alone."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import readout as O
from oracle.operators import TINY, UNIT
from test_gpu_readout import DEV, case, check, on

pytestmark = pytest.mark.gpu


def exact(x, w, b, index, weight, legal, scale, dtype, bias_dtype, chunk=40):
    """Loss, dx, dw, db and their bounds, in float64 on the device: O.loss and O.bounds over chunks of rows, but for sums over the
    columns.  Of those a wave adds 2 ^ 5 or 6 columns as a tree, a lane 1 / 64 of the waves' sums one after the other, and a product
    blocks of 32."""
    x, w, b, scale = x.double(), w.double(), b.double(), scale.double()
    (rows, d), v = x.shape, w.shape[0]
    ax, aw = x.abs(), w.abs()
    f32, u, op = dtype == "float32", O.U, O.OPERAND[dtype]
    wide, tall = aw.amax(1), ax.amax(1)
    n = index.shape[1]
    sums = [torch.zeros(v, d, dtype=torch.float64, device=DEV) for _ in range(3)]
    flat = [torch.zeros(v, dtype=torch.float64, device=DEV) for _ in range(3)]
    out = []
    most = 0.0
    for i in range(0, rows, chunk):
        p = slice(i, i + chunk)
        seen = legal[p].bool()
        z = x[p] @ w.t() + b
        ez = (op + (d + 40) * u) * (ax[p] @ aw.t()) + 4 * u * (z.abs() + b.abs())
        ez_row = torch.where(seen, ez, 0.0).amax(1, keepdim=True)
        z = torch.where(seen, z, -torch.inf)
        top = z.amax(1, keepdim=True)
        top = torch.where(top.isfinite(), top, 0.0)
        gap = torch.where(seen, top - z, 0.0)
        lse = torch.logsumexp(z, 1, keepdim=True)
        at = index[p].long().clamp(min=0)
        a = torch.where((index[p] >= 0) & seen.gather(1, at), weight[p].double(), 0.0)
        share, whole = a.sum(1, keepdim=True), a.abs().sum(1, keepdim=True)
        far = torch.where(a != 0, lse - z.gather(1, at), 0.0)
        loss = (a * far).sum(1)
        e_lse = ez_row + 3 * u * gap.clamp(max=30).amax(1, keepdim=True) + 2.0 ** -22 + (80 + v / 2048) * u + 2.0 ** -21 * np.log2(v + 2.0)
        e_loss = (a.abs() * (ez.gather(1, at) + e_lse + (n + 12) * u * (gap.gather(1, at) + np.log(v) + 1))).sum(1) \
            + whole[:, 0] * (e_lse[:, 0] + 1e-7)
        prob = torch.where(seen & (whole > 0), torch.exp(z - lse), 0.0)
        t = torch.zeros_like(z).scatter_add_(1, at, a)
        sizes = torch.zeros_like(z).scatter_add_(1, at, a.abs())
        g = share * prob - t
        ep = prob * torch.expm1(ez + e_lse + 6 * u * (gap + 1) + 2.0 ** -21)
        if not f32:
            ep += torch.where(t != 0, 0.0, prob * O.STEP * 1.01 + np.exp(-32.0))
        eg = share.abs() * ep + (n + 8) * u * (whole * prob + sizes)
        held = O.HELD[dtype] * (g.abs() + eg) + 4 * u * g.abs() + 1e-38
        s = scale[p].abs()[:, None]
        size, er = g.abs() * s, (eg + held + O.HELD_LEAST[dtype] * whole) * s
        if f32:
            er += O.HELD_LEAST[dtype] * 4 * whole * s * torch.where(wide > 0, wide.max() / wide, 0.0)
        ec = (eg + held) * s
        gs = g * scale[p][:, None]
        e_dx = er @ aw + (op + (v / 32 + 64) * u) * ((size + er) @ aw)
        out.append((loss, gs @ w, e_loss, e_dx))
        sums[0] += gs.t() @ x[p]
        sums[1] += ec.t() @ ax[p] + (op + (rows + 40) * u) * ((size + ec).t() @ ax[p])
        flat[0] += gs.sum(0)
        flat[1] += (eg * s).sum(0) + (rows + 8) * u * size.sum(0)
        flat[2] += size.sum(0)
        most = max(most, float((whole[:, 0] * s[:, 0] * (tall[p] if f32 else 1.0)).max()))
        sums[2] += O.HELD_LEAST[dtype] * 4 * torch.ones_like(g).t() @ (ax[p] / tall[p].clamp(min=1e-300)[:, None] if f32 else ax[p])
    loss, gx, e_loss, e_dx = (torch.cat(p) for p in zip(*out))
    r = lambda e, g, ty: 1.02 * (e + UNIT[ty] * g.abs()) + TINY[ty]
    e_dw = sums[1] + most * sums[2]
    return ((loss, gx, sums[0], flat[0]), (1.02 * e_loss + 1e-30, r(e_dx, gx, dtype), r(e_dw, sums[0], dtype),
                                          r(flat[1], flat[0], bias_dtype)), flat[2])


@pytest.mark.parametrize("dtype,rows,piece,index", [("float32", 400, 320, torch.int32), ("bfloat16", 700, 640, torch.int64)])
def test_two_pieces(dtype, rows, piece, index):
    """2^20 columns: 12 bytes of a float32 logit are 320 rows of 4 GiB, 6 of a 16-bit one 640."""
    from chessfly.readout import Visits, readout_loss, readout_loss_and_grad
    v, d, k = 1 << 20, 4, 3
    g = torch.Generator(device=DEV).manual_seed(rows)
    t = getattr(torch, dtype)
    x = torch.randn(rows, d, generator=g, device=DEV).to(t)
    w = (0.5 * torch.randn(v, d, generator=g, device=DEV)).to(t)
    x[piece + 3], w[1000] = 0.0, 0.0
    b = torch.randn(v, generator=g, device=DEV)
    legal = torch.rand(rows, v, generator=g, device=DEV) < 0.7
    ind = torch.randint(-1, v, (rows, k), generator=g, device=DEV)
    ind[:, 1] = ind[:, 0]                                # the same move twice
    legal.scatter_(1, ind.clamp(min=0), True)
    legal[piece + 5] = False                             # nothing to see, in the second piece
    ind = ind.to(index)
    weight = torch.rand(rows, k, generator=g, device=DEV)
    scale = torch.randn(rows, generator=g, device=DEV)
    scale[::7] = 0
    args = lambda p: (x[p], w, b, Visits(ind[p], weight[p]))
    some = lambda p: dict(legal=legal[p], row_scale=scale[p], grad_scale=2.0)
    loss, grads = readout_loss_and_grad(*args(slice(None)), **some(slice(None)))
    want, most, size = exact(x, w, b, ind, weight, legal, 2 * scale, dtype, "float32")
    for name, a, e, m in zip(("loss", "x", "weight", "bias"), (loss, *grads), want, most):
        off = (a.double() - e).abs()
        assert (off <= m).all(), (name, float((off / m).max()), int((off / m).argmax()))
    # the losses alone keep no logits: their pieces and tiles are others, so their sums' order is too
    assert ((readout_loss(*args(slice(None)), legal, "none").double() - want[0]).abs() <= most[0]).all()
    del want, most
    first, second = (readout_loss_and_grad(*args(p), **some(p)) for p in (slice(0, piece), slice(piece, rows)))
    assert torch.equal(loss, torch.cat([first[0], second[0]])) and torch.equal(grads.x, torch.cat([first[1].x, second[1].x]))
    assert loss[piece + 5] == 0 and not grads.x[piece + 5].any()
    for a, p, q, ty, more in ((grads.weight, first[1].weight, second[1].weight, dtype, 0.0),
                              (grads.bias, first[1].bias, second[1].bias, "float32", 34 * 2.0 ** -24 * size)):
        p, q = p.double(), q.double()
        # each part's rounding and the sum's, and of the bias the order of a piece's sums
        assert ((a.double() - (p + q)).abs() <= 1.02 * UNIT[ty] * (p.abs() + q.abs() + (p + q).abs()) + more + TINY[ty]).all()


def test_more_rows_than_tiles_can_count():
    """2^19 rows and some of few columns."""
    rows, piece = (1 << 19) + 100, 1 << 19
    t = case(rows, 8, 5, "float32", seed=1, k=2, legal=True, index=torch.int32)
    from chessfly.readout import Visits, readout_loss_and_grad
    x, w, b, index, weight, legal = on(*t)
    scale = torch.rand(rows, generator=torch.Generator().manual_seed(2))
    got = readout_loss_and_grad(x, w, b, Visits(index, weight), legal=legal, row_scale=scale.to(DEV))
    check(got, t, "float32", scale.double().numpy())
    alone = readout_loss_and_grad(x[piece:], w, b, Visits(index[piece:], weight[piece:]), legal=legal[piece:],
                                  row_scale=scale[piece:].to(DEV))
    assert torch.equal(got[0][piece:], alone[0]) and torch.equal(got[1].x[piece:], alone[1].x)
