"""GPU tests of a teacher's top logits and of distillation from them against the float64 oracle, at the sizes, masks and
values where they can go wrong.

Tolerances: an exponent z / T - (a log-sum-exp) of a float32 evaluation is off by at most `rounding` (see the oracle).  The
tail is such a sum; the loss moves by its size (sum p |log(p/q)| + 1) times two of them (p's and q's), doubled for the
divergence's own terms; a gradient by its two parts times as much, plus its rounding to the logits' type."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import operators as O

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
NAMES = {torch.float32: "float32", torch.float16: "float16", torch.bfloat16: "bfloat16"}
FLOATS = list(NAMES)
INF = float("inf")


def _logits(rows, cols, seed, dtype=torch.float32, scale=3.0):
    g = torch.Generator().manual_seed(seed)
    return (scale * torch.randn(rows, cols, generator=g)).to(dtype)


def _mask(rows, cols, seed, share):
    g = torch.Generator().manual_seed(seed)
    legal = torch.rand(rows, cols, generator=g) < share
    legal[0] = False                     # a finished game
    if rows > 1:
        legal[1] = True
    return legal


def _np(t):
    return None if t is None else t.double().numpy() if t.is_floating_point() else t.numpy()


def _dev(t):
    return None if t is None else t.to(DEV)


def _check_top(z, k, temperature=1.0, legal=None, zd=None, legal_d=None):
    from chessfly.distill import top_logits
    got = top_logits(_dev(z) if zd is None else zd, k, temperature, _dev(legal) if legal_d is None else legal_d)
    values, index, tail = O.top(_np(z), k, temperature, _np(legal))
    assert np.array_equal(got.index.cpu().numpy(), index)
    assert np.array_equal(got.values.double().cpu().numpy(), values, equal_nan=True)
    t = got.tail.double().cpu().numpy()
    fine = np.isfinite(tail)
    assert np.array_equal(t[~fine], tail[~fine], equal_nan=True)
    assert np.all(np.abs(t[fine] - tail[fine]) <= O.rounding(_np(z), values, temperature))
    return got


def _check_distill(z, teacher, temperature=1.0, legal=None, grad_scale=1.0, row_scale=None, zd=None):
    """Against the oracle: the one-pass call, the loss alone, and autograd."""
    from chessfly.distill import TopLogits, distill_loss, distill_loss_and_grad
    td = TopLogits(*map(_dev, teacher))
    zd = _dev(z) if zd is None else zd
    kw = dict(temperature=temperature, legal=_dev(legal))
    loss, grad = distill_loss_and_grad(zd, td, grad_scale=grad_scale, row_scale=_dev(row_scale), **kw)
    ref, ref_grad, size, parts = O.distill(_np(z), *map(_np, teacher), temperature, _np(legal))
    w = grad_scale * (_np(row_scale)[:, None] if row_scale is not None else 1.0)
    off = O.rounding(_np(z), _np(teacher[0]), temperature)
    _near(loss, ref, 4 * off * size)
    name = NAMES[z.dtype]
    _near(grad, ref_grad * w, (4 * off + 8 * 2.0 ** -24) * np.abs(parts * w)
          + 1.01 * O.UNIT[name] * np.abs(ref_grad * w) + O.TINY[name])
    assert grad.dtype == z.dtype
    alone = distill_loss(zd, td, reduction="none", **kw)
    assert torch.equal(torch.nan_to_num(alone, 7.0), torch.nan_to_num(loss, 7.0))
    leaf = zd.detach().clone().requires_grad_(True)
    up = torch.full((z.shape[0],), float(grad_scale)) * (row_scale if row_scale is not None else 1.0)
    distill_loss(leaf, td, reduction="none", **kw).backward(_dev(up.float()))
    assert torch.equal(torch.nan_to_num(leaf.grad, 7.0), torch.nan_to_num(grad, 7.0)) or row_scale is not None
    return loss, grad


def _near(got, ref, tol):
    got = got.double().cpu().numpy()
    fine = np.isfinite(ref)
    assert np.array_equal(got[~fine], ref[~fine], equal_nan=True)
    off = np.abs(got[fine] - ref[fine])
    tol = np.broadcast_to(tol, ref.shape)[fine]
    assert np.all(off <= tol), float(np.max(off / np.maximum(tol, 1e-300)))


def _teacher(rows, cols, k, seed, temperature, legal=None, tail=True):
    values, index, rest = O.top(_np(_logits(rows, cols, seed)), k, temperature, _np(legal))
    f = lambda a: torch.from_numpy(a.astype(np.float32))
    return f(values), torch.from_numpy(index), f(rest) if tail else None


SIZES = [(1, 1), (2, 2), (3, 3), (3, 31), (2, 33), (4, 64), (3, 65), (5, 257), (3, 1000), (2, 1025), (4, 4168), (2, 5003)]
LONG = [(2, 16384), (2, 16385), (3, 32000), (2, 50257), (2, 65537), (1, 140001), (1, 1 << 20)]


@pytest.mark.parametrize("rows,cols", SIZES)
@pytest.mark.parametrize("k", [1, 2, 7, 32, 218, 256])
@pytest.mark.parametrize("dtype", FLOATS)
def test_top(rows, cols, k, dtype):
    z = _logits(rows, cols, cols + k, dtype)
    _check_top(z, k, 1.5)
    _check_top(z, k, 0.5, _mask(rows, cols, k, 0.3))


@pytest.mark.parametrize("rows,cols", LONG)
@pytest.mark.parametrize("k,dtype", [(1, torch.float32), (64, torch.bfloat16), (256, torch.float16), (40, torch.float32)])
def test_top_of_long_rows(rows, cols, k, dtype):
    _check_top(_logits(rows, cols, cols, dtype), k, 2.0)
    _check_top(_logits(rows, cols, cols, dtype), k, 2.0, _mask(rows, cols, 3, 0.01))


@pytest.mark.parametrize("cols", [40, 300, 4168, 33000, 70000])
@pytest.mark.parametrize("k", [1, 32, 200])
def test_top_of_ties(cols, k):
    """Few different values, or one: the network's policy before its first step gives the same logit for every move."""
    g = torch.Generator().manual_seed(cols)
    z = torch.randint(-2, 3, (6, cols), generator=g).float()
    z[0] = 0.0
    z[1] = -1.5
    z[2] = torch.where(torch.rand(cols, generator=g) < 0.5, 0.0, -0.0)       # zeros of both signs are equal
    z[3, : cols // 2] = 5.0
    z[4, cols - cols // 3:] = 5.0
    _check_top(z, k)
    _check_top(z.half(), k, 1.0, _mask(6, cols, 1, 0.5))
    falling = torch.arange(cols, 0, -1).float().expand(2, -1) / 8
    _check_top(falling.contiguous(), k)
    _check_top(falling.flip(1).contiguous(), k)


@pytest.mark.parametrize("rows", [3, 1030])
@pytest.mark.parametrize("cols", [75, 300, 511, 700, 1024, 1500, 2100])
@pytest.mark.parametrize("k", [60, 256])
def test_top_of_a_large_part_of_the_row(rows, cols, k):
    _check_top(_logits(rows, cols, cols), k, 1.0)
    _check_top(_logits(rows, cols, cols, torch.bfloat16), k, 1.0, _mask(rows, cols, 4, 0.7))


@pytest.mark.parametrize("cols", [37, 4168, 70000])
@pytest.mark.parametrize("dtype", FLOATS)
def test_top_of_odd_values(cols, dtype):
    low = torch.finfo(dtype).min
    z = _logits(8, cols, 3, dtype)
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
    _check_top(z, 4)
    _check_top(z, 30, 1.0, _mask(8, cols, 4, 0.5))


@pytest.mark.parametrize("cols", [4168, 33000, 70000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_top_of_visible_columns_side_by_side(cols, dtype):
    """All that a row shows lies in the columns of one wave: fewer than k, exactly k, and more, on one value and on many."""
    z = _logits(6, cols, 9, dtype)
    legal = torch.zeros(6, cols, dtype=torch.bool)
    for r, n in enumerate([1, 140, 256, 257, 500, 250]):
        legal[r, 16 * r: 16 * r + n] = True
    z[2] = z[5] = 0.75
    for k in (130, 256):
        _check_top(z, k, 1.0, legal)


def test_top_strides_streams_and_no_rows():
    from chessfly.distill import top_logits
    wide = _logits(9, 4300, 7)
    mask = _mask(9, 4303, 8, 0.2)
    _check_top(wide[:, 5:4173], 32, 1.0, mask[:, 3:4171], zd=wide.to(DEV)[:, 5:4173], legal_d=mask.to(DEV)[:, 3:4171])
    half = wide.half()
    _check_top(half[::2, 1:4169], 32, zd=half.to(DEV)[::2, 1:4169])
    _check_top(wide, 9, zd=wide.t().contiguous().to(DEV).t())
    side = torch.cuda.Stream()
    zd = wide.to(DEV)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = top_logits(zd, 32)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, top_logits(zd, 32)))
    assert top_logits(zd[:0], 5).values.shape == (0, 5)
    assert top_logits(zd, 5, tail=False).tail is None


@pytest.mark.parametrize("rows,cols", SIZES)
@pytest.mark.parametrize("k", [1, 7, 32, 218])
@pytest.mark.parametrize("dtype", FLOATS)
def test_distill(rows, cols, k, dtype):
    z = _logits(rows, cols, cols + k, dtype)
    _check_distill(z, _teacher(rows, cols, k, 5, 2.0), 2.0, grad_scale=0.25)
    _check_distill(z, _teacher(rows, cols, k, 5, 1.0, tail=False), 1.0)
    legal = _mask(rows, cols, k, 0.3)
    _check_distill(z, _teacher(rows, cols, k, 5, 0.5, legal), 0.5, legal, row_scale=torch.linspace(0, 2, rows))


@pytest.mark.parametrize("rows,cols", LONG)
@pytest.mark.parametrize("k,dtype", [(1, torch.float32), (64, torch.bfloat16), (256, torch.float16)])
def test_distill_long_rows(rows, cols, k, dtype):
    z = _logits(rows, cols, cols, dtype)
    _check_distill(z, _teacher(rows, cols, k, 5, 2.0), 2.0)
    legal = _mask(rows, cols, 3, 0.01)
    _check_distill(z, _teacher(rows, cols, k, 5, 1.0, legal, tail=False), 1.0, legal)


@pytest.mark.parametrize("cols", [37, 4168, 70000])
@pytest.mark.parametrize("dtype", FLOATS)
def test_distill_odd_values(cols, dtype):
    low = torch.finfo(dtype).min
    values, index, tail = _teacher(12, cols, 6, 3, 1.0)
    z = _logits(12, cols, 4, dtype)
    z[0] = -INF                                  # the student sees nothing
    z[1] = low
    z[2, ::3] = low
    z[3] = -INF
    z[3, index[3, 0].item()] = 1.0               # nothing but one listed move: the rest has no column, others -inf
    z[4, index[4, 1].item()] = -INF              # the teacher's move is impossible: infinite loss, finite gradient
    z[5, (index[5, 0].item() + 1) % cols] = float("nan")
    index[6] = -1                                # nothing listed: the tail alone
    index[7, 1:] = -1                            # padding in the middle and at the end
    index[8, 0], index[8, 2] = -1, -5
    values[9, 3:] = -INF                         # listed, of no probability
    tail[10] = -INF
    z[11] += 40.0 if dtype == torch.float32 else 0.0
    _check_distill(z, (values, index, tail))
    index[6] = -1
    _check_distill(z, (values, index, None), 2.0)


def test_distill_bad_lists_are_nan_and_stay_in_their_row():
    from chessfly.distill import TopLogits, distill_loss_and_grad
    values, index, tail = _teacher(5, 300, 6, 3, 1.0)
    z = _logits(5, 300, 4)
    index[1, 2] = 300
    index[2, 5] = index[2, 0]
    index[3, 1] = 2 ** 31 - 1
    loss, grad = _check_distill(z, (values, index, tail))
    assert torch.isnan(loss).tolist() == [False, True, True, True, False]
    keep = torch.tensor([0, 4])
    ref = distill_loss_and_grad(z[keep].to(DEV), TopLogits(values[keep].to(DEV), index[keep].to(DEV), tail[keep].to(DEV)))
    assert torch.equal(loss[keep], ref[0]) and torch.equal(grad[keep], ref[1])


def test_a_small_divergence_keeps_its_digits():
    """A student near its teacher: the loss is of second order in the difference, the logits' rounding of first."""
    from chessfly.distill import TopLogits, distill_loss
    t = _logits(16, 4168, 1)
    z = t + 1e-2 * _logits(16, 4168, 2, scale=1.0)
    values, index, tail = O.top(_np(t), 32, 1.0)
    f = lambda a: torch.from_numpy(a.astype(np.float32))
    teacher = (f(values), torch.from_numpy(index), f(tail))
    ref, _, _, _ = O.distill(_np(z), *map(_np, teacher), 1.0)
    got = distill_loss(z.to(DEV), TopLogits(*map(_dev, teacher)), reduction="none").double().cpu().numpy()
    assert ref.max() < 1e-4
    # an exponent off by e moves the loss by sum |p - q| e <= sqrt(2 loss) e (Pinsker), and by e^2
    e = 2 * O.rounding(_np(z), values, 1.0)
    assert np.all(np.abs(got - ref) <= np.sqrt(2 * ref) * e + e * e + 8 * 2.0 ** -24 * np.sqrt(2 * ref) * 0.1 + 1e-12)


def test_gradient_against_differences():
    """The loss along a direction v, (L(z + e v) - L(z - e v)) / 2e: the loss's float32 error over e, plus e^2 / 6 of a third
    derivative, which is at most 2 / T (max |v|)^3 for a log-sum-exp."""
    from chessfly.distill import TopLogits, distill_loss, distill_loss_and_grad
    z, T, e = _logits(8, 500, 1), 2.0, 2.0 ** -5
    teacher = _teacher(8, 500, 20, 5, T)
    td = TopLogits(*map(_dev, teacher))
    _, grad = distill_loss_and_grad(z.to(DEV), td, T)
    g = torch.Generator().manual_seed(3)
    _, _, size, _ = O.distill(_np(z), *map(_np, teacher), T)
    for _ in range(4):
        v = torch.sign(torch.randn(8, 500, generator=g))
        up, down = (distill_loss((z + s * e * v).to(DEV), td, T, reduction="none").double().cpu().numpy() for s in (1, -1))
        want = (grad.double().cpu() * v).sum(1).numpy()
        tol = 4 * O.rounding(_np(z), _np(teacher[0]), T) * size / e + e * e / 6 * 2 / T * 2 ** 3 + e * 2.0 ** -20
        assert np.all(np.abs((up - down) / (2 * e) - want) <= tol)


@pytest.mark.parametrize("reduction", ["mean", "sum"])
def test_autograd_reductions_and_shared_logits(reduction):
    """The loss of logits that a broadcast made: their gradients add up."""
    from chessfly.distill import TopLogits, distill_loss, distill_loss_and_grad
    teacher = TopLogits(*map(_dev, _teacher(6, 700, 9, 5, 1.0)))
    z = _logits(1, 700, 2).to(DEV).requires_grad_(True)
    distill_loss(z.expand(6, -1), teacher, reduction=reduction).backward()
    scale = 1 / 6 if reduction == "mean" else 1.0
    _, grad = distill_loss_and_grad(z.detach().expand(6, -1).contiguous(), teacher, grad_scale=scale)
    assert torch.allclose(z.grad, grad.sum(0, keepdim=True), rtol=1e-5, atol=1e-7)


def test_distill_strides_streams_graph_and_no_rows():
    from chessfly.distill import TopLogits, distill_loss, distill_loss_and_grad, top_logits
    wide = _logits(9, 4301, 7)
    teacher = _teacher(9, 4168, 32, 5, 1.0)
    for t in (wide, wide.half(), wide.bfloat16()):
        _check_distill(t[:, 5:4173], teacher, zd=t.to(DEV)[:, 5:4173])
    wide2 = _logits(18, 4168, 7)
    _check_distill(wide2[::2], teacher, zd=wide2.to(DEV)[::2])
    _check_distill(wide2[:9], teacher, zd=wide2[:9].t().contiguous().to(DEV).t())
    td = TopLogits(*map(_dev, teacher))
    z = wide[:, :4168].contiguous().to(DEV)
    ref = distill_loss_and_grad(z, td)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = distill_loss_and_grad(z, td)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        labels = top_logits(z, 32)
        out = distill_loss_and_grad(z, TopLogits(labels.values, labels.index, labels.tail))
    for seed in range(3):
        z.copy_(_logits(9, 4168, 30 + seed))
        graph.replay()
        torch.cuda.synchronize()
        now = top_logits(z, 32)
        again = distill_loss_and_grad(z, now)
        assert all(torch.equal(a, b) for a, b in zip(labels, now))
        assert torch.equal(out[0], again[0]) and torch.equal(out[1], again[1])
    none = TopLogits(td.values[:0], td.index[:0], td.tail[:0])
    loss, grad = distill_loss_and_grad(z[:0], none)
    assert loss.shape == (0,) and grad.shape == (0, 4168)
    assert distill_loss(z[:0], none, reduction="none").shape == (0,)


@pytest.mark.parametrize("rows,cols,k", [(64, 4168, 32), (9, 4168, 218), (1100, 600, 20), (3, 70000, 100)])
def test_results_repeat_bit_for_bit(rows, cols, k):
    """The order in which workgroups and lanes meet in LDS leaves no trace."""
    from chessfly.distill import distill_loss_and_grad, top_logits
    z, t = _logits(rows, cols, 1).to(DEV), _logits(rows, cols, 2).to(DEV)
    first = top_logits(t, k, 2.0)
    ref = distill_loss_and_grad(z, first, 2.0)
    for _ in range(5):
        again = top_logits(t, k, 2.0)
        assert all(torch.equal(a, b) for a, b in zip(first, again))
        assert all(torch.equal(a, b) for a, b in zip(ref, distill_loss_and_grad(z, again, 2.0)))


def test_offsets_past_32_bits():
    """Rows over 2^31 elements apart."""
    from chessfly.distill import TopLogits, distill_loss_and_grad, top_logits
    cols, apart = 4168, 1_150_000_000
    big = torch.empty(2 * apart + cols, dtype=torch.float16, device=DEV)
    zd = big.as_strided((3, cols), (apart, 1))
    z = _logits(3, cols, 3, torch.float16)
    zd.copy_(z)
    teacher = TopLogits(*map(_dev, _teacher(3, cols, 32, 5, 1.0)))
    assert all(torch.equal(a, b) for a, b in zip(top_logits(zd, 32), top_logits(z.to(DEV), 32)))
    for a, b in zip(distill_loss_and_grad(zd, teacher), distill_loss_and_grad(z.to(DEV), teacher)):
        assert torch.equal(a, b)


def test_refusals():
    from chessfly.distill import TopLogits, distill_loss, distill_loss_and_grad, top_logits
    z = torch.zeros(3, 12, device=DEV)
    v, i, t = torch.zeros(3, 4, device=DEV), torch.zeros(3, 4, dtype=torch.int32, device=DEV), torch.zeros(3, device=DEV)
    legal = torch.ones(3, 12, dtype=torch.bool, device=DEV)
    for call in (lambda: top_logits(z, 0), lambda: top_logits(z, 257), lambda: top_logits(z.double(), 3),
                 lambda: top_logits(z[0], 3), lambda: top_logits(z, 3, legal=legal[:2]),
                 lambda: top_logits(z, 3, legal=legal.cpu()), lambda: top_logits(z, 3, legal=legal.float()),
                 lambda: top_logits(z, 3, temperature=0.0), lambda: distill_loss(z, (v, i.long(), t)),
                 lambda: distill_loss(z, (v[:2], i, t)), lambda: distill_loss(z, (v, i[:, :2], t)),
                 lambda: distill_loss(z, (v, i, t.half())), lambda: distill_loss(z, (v, i, t), reduction="batch"),
                 lambda: distill_loss(z, (v, i, t), temperature=-1.0), lambda: distill_loss(z.to(torch.int8), (v, i, t)),
                 lambda: distill_loss(z, (v.cpu(), i, t)), lambda: distill_loss(z[:, :0], (v, i, t)),
                 lambda: distill_loss_and_grad(z, TopLogits(v, i, t), row_scale=t[:2])):
        with pytest.raises(RuntimeError):
            call()
