"""GPU tests of the read-out loss and its gradients against the float64 oracle, element by element within the roundings that the
kernels make (oracle/readout.py)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import readout as O

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
SIZES = [(1, 1, 1), (1, 70, 333), (2, 5, 3), (3, 33, 31), (16, 32, 32), (17, 31, 33), (31, 65, 129), (33, 64, 128), (64, 100, 257),
         (65, 513, 300), (130, 257, 1000), (257, 40, 520), (300, 1, 1), (259, 33, 31), (310, 97, 129), (385, 600, 200), (513, 31, 2000)]


FEW, MANY = 40, 280    # rows that take the kernels of few rows, and those of many, whatever the type


def case(rows, d, v, dtype, seed=0, k=1, legal=False, bias="own", index=torch.int64, spread=2.0):
    """Tensors of one call; None where there is none.  Every fourth row's targets hold -1s, every seventh row sees nothing."""
    g = torch.Generator().manual_seed(seed)
    t = TYPES[dtype]
    x = torch.randn(rows, d, generator=g).to(t)
    w = (spread * torch.randn(v, d, generator=g) / d ** 0.5).to(t)
    b = {"own": t, "float32": torch.float32, None: None}[bias]
    b = torch.randn(v, generator=g).to(b) if b is not None else None
    ind = torch.randint(0, v, (rows, k), generator=g)
    ind[::4] = torch.where(torch.rand(ind[::4].shape, generator=g) < 0.5, -1, ind[::4])
    weight = torch.rand(rows, k, generator=g) if k > 1 else None
    mask = None
    if legal:
        mask = torch.rand(rows, v, generator=g) < 0.4
        mask.scatter_(1, ind.clamp(min=0), True)
        mask[3::7] = False
    return x, w, b, (ind if k > 1 else ind[:, 0]).to(index), weight, mask


def on(*tensors):
    return [None if t is None else t.to(DEV) for t in tensors]


def call(x, w, b, index, weight, legal, **kw):
    from chessfly.readout import Visits, readout_loss_and_grad
    x, w, b, index, weight, legal = on(x, w, b, index, weight, legal)
    return readout_loss_and_grad(x, w, b, index if weight is None else Visits(index, weight), legal=legal, **kw)


def numpy(*tensors):
    return [None if t is None else t.double().numpy() if t.is_floating_point() else t.numpy() for t in tensors]


def check(got, tensors, dtype, scale=None):
    x, w, b, index, weight, legal = numpy(*tensors)
    bt = None if tensors[2] is None else str(tensors[2].dtype)[6:]
    want = O.loss(x, w, b, index, weight, legal, scale)
    most = O.bounds(x, w, b, index, dtype, weight, legal, scale, bt)
    loss, grads = got
    assert loss.dtype == torch.float32 and (grads.bias is None) == (b is None)
    for name, a, e, m in zip(("loss", "x", "weight", "bias"), (loss, *grads), want, most):
        if a is None:
            continue
        off = np.abs(a.double().cpu().numpy() - e)
        assert (off <= m).all(), (name, float((off / m).max()), np.unravel_index(np.argmax(off / m), off.shape))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,d,v", SIZES)
def test_one_target(rows, d, v, dtype):
    t = case(rows, d, v, dtype, seed=rows)
    check(call(*t, grad_scale=0.5), t, dtype, np.full(rows, 0.5))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,d,v", SIZES)
@pytest.mark.parametrize("k", [5, 70])
def test_visits_over_legal_moves(rows, d, v, dtype, k):
    """Lists longer than the columns list them twice: their weights add up."""
    t = case(rows, d, v, dtype, seed=7 * rows + k, k=k, legal=True, bias="float32", index=torch.int32)
    g = torch.Generator().manual_seed(1)
    scale = torch.randn(rows, generator=g)
    scale[::5] = 0
    check(call(*t, grad_scale=2.0, row_scale=scale.to(DEV)), t, dtype, 2.0 * scale.double().numpy())


@pytest.mark.parametrize("rows", [FEW, MANY])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_weights_of_both_signs_without_bias(dtype, rows):
    t = list(case(rows, 50, 60, dtype, k=4, bias=None))
    t[4] = torch.randn(rows, 4, generator=torch.Generator().manual_seed(3)) * 100
    check(call(*t), t, dtype)


@pytest.mark.parametrize("rows", [20, 479])
def test_one_column_with_weights_of_both_signs(rows):
    """The gradient is 0 but for the weights' sums, taken in two orders."""
    t = list(case(rows, 17, 1, "bfloat16", k=70, bias="float32", seed=rows))
    t[4] -= 0.5
    check(call(*t, grad_scale=0.3), t, "bfloat16", np.full(rows, float(np.float32(0.3))))


@pytest.mark.parametrize("rows", [FEW, MANY])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_confident_rows(dtype, rows):
    """Logits of up to some 100, whose softmax is all but 0 and 1."""
    t = case(rows, 64, 200, dtype, seed=5, k=3, spread=30.0)
    check(call(*t), t, dtype)


@pytest.mark.parametrize("rows", [FEW, MANY])
def test_rows_and_weights_of_very_different_size(rows):
    """float32 rows are multiplied by units of their own."""
    x, w, b, index, weight, legal = case(rows, 40, 90, "float32", seed=9, k=3)
    g = torch.Generator().manual_seed(2)
    x = x * 10.0 ** torch.randint(-6, 1, (rows, 1), generator=g)
    w = w * 10.0 ** torch.randint(-6, 1, (90, 1), generator=g)
    t = (x, w, b, index, weight, legal)
    check(call(*t), t, "float32")
    for size in (1e18, 1e30):
        t = (x * size, w / size, b, index, weight, legal)
        check(call(*t), t, "float32")


@pytest.mark.parametrize("rows", [37, 277])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_strides(dtype, rows):
    """Rows apart, columns apart, a transposed weight, every second target, a mask that is a part of a larger one."""
    from chessfly.readout import Visits, readout_loss_and_grad
    x, w, b, index, weight, legal = on(*case(rows, 70, 150, dtype, k=4, legal=True))
    want = readout_loss_and_grad(x, w, b, Visits(index, weight), legal=legal)
    wide = torch.zeros(rows, 101, dtype=x.dtype, device=DEV)
    wide[:, 3:73] = x
    apart = torch.zeros(150, 140, dtype=x.dtype, device=DEV)
    apart[:, ::2] = w
    large = torch.zeros(rows + 3, 155, dtype=torch.bool, device=DEV)
    large[1:rows + 1, 2:152] = legal
    idx = torch.zeros(rows, 8, dtype=index.dtype, device=DEV)
    idx[:, ::2] = index
    bb = torch.zeros(300, dtype=b.dtype, device=DEV)
    bb[::2] = b
    variants = [(wide[:, 3:73], w, b, index, weight, legal), (x, w.t().contiguous().t(), b, index, weight, legal),
                (x, apart[:, ::2], bb[::2], idx[:, ::2], weight.t().contiguous().t(), large[1:rows + 1, 2:152]),
                (x, w, b, index, weight, legal.to(torch.uint8))]
    for x_, w_, b_, i_, a_, l_ in variants:
        got = readout_loss_and_grad(x_, w_, b_, Visits(i_, a_), legal=l_)
        assert torch.equal(got[0], want[0]) and all(torch.equal(p, q) for p, q in zip(got[1], want[1]))


@pytest.mark.parametrize("rows", [20, 300])
def test_broadcast_rows(rows):
    """One row for all, and one mask: strides of 0."""
    from chessfly.readout import readout_loss_and_grad
    x, w, b, index, _, legal = on(*case(rows, 33, 47, "float32", legal=True))
    legal[0] = True
    a = readout_loss_and_grad(x[:1].expand(rows, 33), w, b, index, legal=legal[:1].expand(rows, 47))
    e = readout_loss_and_grad(x[:1].repeat(rows, 1), w, b, index, legal=legal[:1].repeat(rows, 1))
    assert torch.equal(a[0], e[0]) and all(torch.equal(p, q) for p, q in zip(a[1], e[1]))


@pytest.mark.parametrize("rows", [FEW, MANY])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_a_row_that_is_not_finite_stays_its_own(dtype, rows):
    t = list(case(rows, 50, 60, dtype, k=3))
    t[3] = t[3].abs()
    want = call(*t)
    for bad in (float("nan"), float("inf")):
        x = t[0].clone()
        x[11, 5] = bad
        loss, grads = call(x, *t[1:])
        others = torch.arange(rows) != 11
        assert loss[11].isnan() and grads.x[11].isnan().any()
        assert torch.equal(loss[others], want[0][others]) and torch.equal(grads.x[others], want[1].x[others])


@pytest.mark.parametrize("rows", [FEW, MANY])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_rows_left_out_may_hold_anything(dtype, rows):
    t = list(case(rows, 50, 60, dtype, k=3))
    t[3][10:14] = -1
    want = call(*t)
    x = t[0].clone()
    x[10:12], x[12:14] = float("nan"), float("inf")
    got = call(x, *t[1:])
    assert (got[0][10:14] == 0).all() and (got[1].x[10:14] == 0).all()
    assert torch.equal(got[0], want[0]) and all(torch.equal(p, q) for p, q in zip(got[1], want[1]))


@pytest.mark.parametrize("rows", [FEW, MANY])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_hidden_columns_may_hold_anything(dtype, rows):
    """NaN and infinite biases of columns that no row sees; a type's lowest value in place of a mask."""
    x, w, b, index, weight, legal = case(rows, 50, 60, dtype, k=3, legal=True)
    hidden = torch.arange(60) % 5 == 2
    legal = legal & ~hidden
    want = call(x, w, b, index, weight, legal)
    for bad in (float("nan"), float("inf"), -float("inf"), 1e4):
        got = call(x, w, torch.where(hidden, torch.tensor(bad, dtype=b.dtype), b), index, weight, legal)
        assert torch.equal(got[0], want[0]) and all(torch.equal(p, q) for p, q in zip(got[1], want[1]))
    seen = ~hidden[index.clamp(min=0)]
    weight = torch.where(seen, weight, 0.0)
    want = call(x, w, b, index, weight, (~hidden).expand(rows, 60))
    got = call(x, w, torch.where(hidden, torch.tensor(torch.finfo(b.dtype).min, dtype=b.dtype), b), index, weight, None)
    assert torch.equal(got[0], want[0]) and all(torch.equal(p, q) for p, q in zip(got[1], want[1]))


@pytest.mark.parametrize("rows", [FEW, MANY])
def test_targets_past_the_columns(rows):
    t = list(case(rows, 50, 60, "float32", k=3))
    want = call(*t)
    t[3][7, 1] = 60
    t[3][9, 0] = 2 ** 40
    loss, grads = call(*t)
    bad = torch.isin(torch.arange(rows), torch.tensor([7, 9]))
    assert loss[bad].isnan().all() and grads.x[bad].isnan().all()
    assert torch.equal(loss[~bad], want[0][~bad]) and torch.equal(grads.x[~bad], want[1].x[~bad])


def test_infinite_losses_follow_the_formula():
    """A target at -inf has an infinite loss and the gradient of its weight."""
    x, w, b, index, _, _ = case(4, 8, 6, "float32")
    index, b = torch.tensor([0, 1, 2, 1]), b.clone()
    b[1] = -float("inf")
    loss, grads = call(x, w, b, index, None, None)
    assert loss.tolist()[1] == float("inf") and loss.tolist()[3] == float("inf") and loss[[0, 2]].isfinite().all()
    assert grads.x.isfinite().all() and abs(float(grads.bias[1]) + 2) < 1e-6


def test_no_rows():
    from chessfly.readout import readout_loss, readout_loss_and_grad
    x, w = torch.zeros(0, 9, device=DEV), torch.randn(7, 9, device=DEV)
    t = torch.zeros(0, dtype=torch.int64, device=DEV)
    loss, grads = readout_loss_and_grad(x, w, torch.zeros(7, device=DEV), t)
    assert loss.shape == (0,) and grads.x.shape == (0, 9) and not grads.weight.any() and not grads.bias.any()
    assert readout_loss(x, w, None, t, reduction="sum") == 0


def test_rows_in_pieces():
    """2^20 columns: 300 rows' logits fit no piece.  Against the formula in float64, each gradient within the roundings of u and
    of itself, the steps of the logits that wait, and float32 sums of as many steps as the columns or rows have blocks of 32."""
    from chessfly.readout import readout_loss_and_grad
    v, d, rows = 1 << 20, 4, 700
    g = torch.Generator(device=DEV).manual_seed(1)
    x, w = (torch.randn(n, d, generator=g, device=DEV).half() for n in (rows, v))
    b, t = torch.randn(v, generator=g, device=DEV), torch.randint(0, v, (rows,), generator=g, device=DEV)
    loss, grads = readout_loss_and_grad(x, w, b, t)
    want, gx = torch.zeros_like(loss, dtype=torch.float64), torch.zeros(rows, d, dtype=torch.float64, device=DEV)
    size = torch.zeros_like(gx)
    gw, gw_size, gb = torch.zeros(v, d, dtype=torch.float64, device=DEV), torch.zeros(v, d, dtype=torch.float64, device=DEV), 0.0
    for i in range(0, rows, 100):
        p = slice(i, i + 100)
        z = x[p].double() @ w.double().t() + b.double()
        want[p] = torch.logsumexp(z, 1) - z.gather(1, t[p, None])[:, 0]
        u = torch.softmax(z, 1)
        u.scatter_add_(1, t[p, None], torch.full((100, 1), -1.0, dtype=torch.float64, device=DEV))
        gx[p], size[p] = u @ w.double(), u.abs() @ w.double().abs()
        gw += u.t() @ x[p].double()
        gw_size += u.abs().t() @ x[p].double().abs()
        gb = gb + u.sum(0)
    assert ((loss - want).abs() <= 1e-5 * want).all()
    off = lambda a, e, s, n: ((a.double() - e).abs() / ((2.0 ** -11 + 2.0 ** -13 + (n / 32 + 64) * 2.0 ** -24) * s
                                                        + 2.0 ** -11 * e.abs() + 2.0 ** -24)).max()
    assert off(grads.x, gx, size, v) <= 1 and off(grads.weight, gw, gw_size, rows) <= 1
    assert ((grads.bias - gb).abs() <= 2.0 ** -9 * (gb.abs() + 2 * torch.bincount(t, minlength=v))).all()


@pytest.mark.parametrize("rows", [50, 300])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_autograd(dtype, rows):
    """The gradients of readout_loss are those of readout_loss_and_grad, for the leaves that want one."""
    from chessfly.readout import Visits, readout_loss
    t = case(rows, 33, 70, dtype, k=3, legal=True)
    x, w, b, index, weight, legal = on(*t)
    loss, grads = call(*t, grad_scale=1 / rows)
    for wants in ((1, 1, 1), (1, 0, 0), (0, 1, 0), (0, 0, 1)):
        leaves = [p.clone().requires_grad_(bool(n)) for p, n in zip((x, w, b), wants)]
        out = readout_loss(*leaves, Visits(index, weight), legal)
        assert torch.equal(out, loss.mean())
        out.backward()
        for leaf, n, e in zip(leaves, wants, grads):
            assert (leaf.grad is not None) == bool(n)
            # the upstream gradient is 1 / rows rounded to float32 there and here
            if n:
                assert torch.equal(leaf.grad, e)
    with torch.no_grad():
        assert not readout_loss(x.requires_grad_(), w, b, Visits(index, weight), legal).requires_grad


def test_autograd_by_rows_and_shared_leaves():
    """Each row's upstream gradient; a weight used twice gets both shares; no second derivative, no forward mode."""
    from torch.autograd import forward_ad
    from chessfly.readout import readout_loss
    t = case(30, 20, 40, "float32")
    x, w, b, index, _, _ = on(*t)
    up = torch.randn(30, device=DEV)
    _, grads = call(*t, row_scale=up)
    w = w.requires_grad_()
    readout_loss(x, w, b, index, reduction="none").backward(up)
    assert torch.equal(w.grad, grads.weight)
    w.grad = None
    (readout_loss(x, w, b, index, reduction="none") + readout_loss(x, w, b, index, reduction="none")).backward(up)
    assert torch.equal(w.grad, 2 * grads.weight)
    (g,) = torch.autograd.grad(readout_loss(x, w, b, index), w, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    with forward_ad.dual_level(), pytest.raises(RuntimeError):
        readout_loss(forward_ad.make_dual(x, torch.ones_like(x)), w.detach(), b, index)


@pytest.mark.parametrize("rows", [3, 200, 400])
def test_in_a_graph(rows):
    """Captured with its workspace and replayed between eager calls."""
    from chessfly.readout import readout_loss
    x, w, b, index, _, legal = on(*case(rows, 65, 130, "float32", legal=True))
    leaves = [t.requires_grad_() for t in (x, w, b)]
    torch.autograd.grad(readout_loss(*leaves, index, legal), leaves)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = readout_loss(*leaves, index, legal)
        grads = torch.autograd.grad(loss, leaves)
    for seed in range(4):
        g = torch.Generator().manual_seed(seed)
        with torch.no_grad():
            for t in leaves:
                t.copy_(torch.randn(t.shape, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        e = readout_loss(*leaves, index, legal)
        assert torch.equal(loss, e)
        assert all(torch.equal(p, q) for p, q in zip(grads, torch.autograd.grad(e, leaves)))


def test_a_capture_beside_an_eager_graph_of_the_same_leaves_is_refused():
    """Its backward pass would wait for the eager graph's stream, outside the capture."""
    from chessfly.readout import readout_loss
    x, w, b, index, _, _ = on(*case(9, 12, 20, "float32"))
    w.requires_grad_()
    alive = readout_loss(x, w, b, index)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="still alive"):
        with torch.cuda.graph(graph):
            readout_loss(x, w, b, index)
    (eager,) = torch.autograd.grad(alive, w)
    del alive
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        # used twice in one capture: the second use finds the first one's node
        grad = torch.autograd.grad(readout_loss(x, w, b, index) + readout_loss(x, w, b, index), w)[0]
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(grad, 2 * eager)


@pytest.mark.parametrize("rows", [60, 500])
def test_streams_and_repeats(rows):
    """The same bits on another stream and on every call."""
    from chessfly.readout import Visits, readout_loss_and_grad
    x, w, b, index, weight, legal = on(*case(rows, 300, 700, "bfloat16", k=4, legal=True))
    want = readout_loss_and_grad(x, w, b, Visits(index, weight), legal=legal)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(readout_loss_and_grad(x, w, b, Visits(index, weight), legal=legal))
    torch.cuda.synchronize()
    for loss, grads in got:
        assert torch.equal(loss, want[0]) and all(torch.equal(p, q) for p, q in zip(grads, want[1]))


def test_refuses():
    from chessfly.readout import Visits, readout_loss, readout_loss_and_grad
    x, w, b, index, weight, legal = on(*case(6, 5, 4, "float32", k=2, legal=True))
    one = index[:, 0]
    bad = [(x[0], w, b, one), (x, w[:, :3], b, one), (x, w.half(), b, one), (x.int(), w.int(), b, one), (x, w, b[:2], one),
           (x, w, b.half(), one), (x, w, b, one[:3]), (x, w, b, one.float()), (x, w, b, index), (x, w, b, Visits(index, weight.double())),
           (x, w, b, Visits(index, weight[:, :1])), (x, w, b, Visits(index[:, :0], weight[:, :0])), (x, w, b, Visits(one, weight)),
           (x, w, b, one.cpu()), (x, w.cpu(), b, one), (x[:, :0], w[:, :0], b, one),
           (x, w, b, Visits(index.repeat(1, 600), weight.repeat(1, 600)))]
    for args in bad:
        with pytest.raises(RuntimeError):
            readout_loss(*args)
        with pytest.raises(RuntimeError):
            readout_loss_and_grad(*args)
    for mask in (legal[:, :2], legal.float(), legal.cpu()):
        with pytest.raises(RuntimeError):
            readout_loss(x, w, b, one, mask)
    with pytest.raises(RuntimeError, match="row_scale"):
        readout_loss_and_grad(x, w, b, one, row_scale=torch.ones(5, device=DEV))
