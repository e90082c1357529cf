"""GPU tests of the 8-bit dense map against the float64 oracle: quantised values and scales bit for bit, products within the
roundings of the scaling (integer sums are exact)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import operators as O

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
NAMES = {torch.float32: "float32", torch.float16: "float16", torch.bfloat16: "bfloat16"}
FLOATS = list(NAMES)


def _x(rows, k, seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, k, generator=g) * torch.logspace(-2, 2, rows)[:, None]).to(dtype)


def _weight(n, k, seed, bias=True):
    g = torch.Generator().manual_seed(seed)
    w = torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int8)
    return w, torch.rand(n, generator=g) + 0.01, torch.randn(n, generator=g) if bias else None


def _check(y, q, s, w, t, b, dtype):
    ref, bound = O.int8_linear(q, s, w.numpy(), t.numpy(), None if b is None else b.numpy())
    bound = bound + O.UNIT[NAMES[dtype]] * np.abs(ref) * 1.01 + O.TINY[NAMES[dtype]]
    got = y.double().cpu().numpy()
    assert y.dtype == dtype and np.array_equal(np.isnan(got), np.isnan(ref))
    fine = np.abs(ref) <= torch.finfo(dtype).max       # what passes the type's range rounds to an infinity
    assert np.array_equal(got[~fine], np.sign(ref[~fine]) * np.inf, equal_nan=True)
    off = np.abs(got - ref)[fine]
    assert np.all(off <= bound[fine]), float(np.max(off / bound[fine]))


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("rows,k", [(1, 1), (3, 15), (2, 16), (5, 17), (16, 64), (17, 333), (4, 2333), (7, 5000)])
def test_quantised_rows_are_the_definition(rows, k, dtype):
    from chessfly.int8 import quantize_rows
    x = _x(rows, k, rows + k, dtype)
    q, s = quantize_rows(x.to(DEV))
    rq, rs = O.quantize(x.float().numpy())
    assert np.array_equal(s.cpu().numpy(), rs) and np.array_equal(q.cpu().numpy(), rq)


def test_quantised_rows_at_the_edges():
    from chessfly.int8 import Int8Linear, quantize_rows
    x = _x(9, 70, 1)
    x[0] = 0
    x[1, 3] = float("inf")
    x[2, 69] = float("nan")
    x[3, 0] = -float("inf")
    x[4] *= 1e-38                      # subnormal throughout
    x[5, 7] = -3.4028234663852886e38   # the type's lowest value
    x[6] = 2.0 ** -119
    x[7] = -0.0
    q, s = quantize_rows(x.to(DEV))
    rq, rs = O.quantize(x.numpy())
    assert np.array_equal(s.cpu().numpy(), rs, equal_nan=True) and np.array_equal(q.cpu().numpy(), rq)
    w, t, b = _weight(33, 70, 2)
    _check(Int8Linear(w.to(DEV), t.to(DEV), b.to(DEV))(x.to(DEV)), rq, rs, w, t, b, torch.float32)


@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 33, 64, 65, 127, 129, 300])
@pytest.mark.parametrize("n,k", [(1, 1), (3, 2333), (16, 64), (65, 63), (130, 129), (515, 838)])
def test_product(rows, n, k):
    from chessfly.int8 import Int8Linear
    x = _x(rows, k, rows)
    w, t, b = _weight(n, k, n + k, bias=n % 2 == 1)
    y = Int8Linear(w.to(DEV), t.to(DEV), None if b is None else b.to(DEV))(x.to(DEV))
    _check(y, *O.quantize(x.numpy()), w, t, b, torch.float32)


@pytest.mark.parametrize("rows", [1, 21, 517])
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("out", FLOATS)
def test_product_types(rows, dtype, out):
    from chessfly.int8 import Int8Linear
    x = _x(rows, 205, 5, dtype)
    w, t, b = _weight(301, 205, 6)
    y = Int8Linear(w.to(DEV), t.to(DEV) / 100, b.to(DEV))(x.to(DEV), out_dtype=out)
    _check(y, *O.quantize(x.float().numpy()), w, t / 100, b, out)


# Few rows are quantised in the product itself: each count of rows' blocks, a row's length and the channels on both sides
# of where that ends.
@pytest.mark.parametrize("rows", [1, 8, 9, 16, 17, 31, 32, 33])
@pytest.mark.parametrize("n,k,dtype", [(70, 3050, torch.float32), (70, 3050, torch.float16), (70, 3090, torch.bfloat16),
                                       (8190, 100, torch.float16), (8210, 100, torch.float32)])
def test_few_rows(rows, n, k, dtype):
    from chessfly.int8 import Int8Linear
    x = _x(rows, k, rows + 1, dtype)
    w, t, b = _weight(n, k, rows + n, bias=rows % 2 == 1)
    y = Int8Linear(w.to(DEV), t.to(DEV), None if b is None else b.to(DEV))(x.to(DEV))
    _check(y, *O.quantize(x.float().numpy()), w, t, b, torch.float32)


@pytest.mark.parametrize("rows,n,k", [(1, 4168, 2333), (21, 4168, 2333), (250, 4168, 2333), (1120, 4168, 2333),
                                      (517, 17937, 838), (2100, 1030, 700)])
def test_product_at_full_size(rows, n, k):
    from chessfly.int8 import Int8Linear
    x = _x(rows, k, 9)
    w, t, b = _weight(n, k, 10)
    y = Int8Linear(w.to(DEV), t.to(DEV), b.to(DEV))(x.to(DEV))
    q, s = O.quantize(x.numpy())
    # a sample of rows, and every row against the float64 product on the device
    _check(y[: min(rows, 40)], q[:40], s[:40], w, t, b, torch.float32)
    acc = torch.from_numpy(q).to(DEV).double() @ w.to(DEV).double().t()
    ref = acc * (torch.from_numpy(s).to(DEV).double()[:, None] * t.to(DEV).double()) + b.to(DEV).double()
    off = (y.double() - ref).abs()
    assert bool((off <= 4 * 2.0 ** -24 * ((ref - b.to(DEV).double()).abs() + b.to(DEV).double().abs())).all())


def test_rows_in_8_bits_and_the_largest_sums():
    """int8 rows with their scales; every product at its largest, so the sums reach 128 * 128 * k."""
    from chessfly.int8 import Int8Linear
    k = 130000
    q = torch.full((3, k), -128, dtype=torch.int8)
    q[1] = 127
    w = torch.full((5, k), -128, dtype=torch.int8)
    w[2] = 127
    s, t = torch.tensor([1.0, 0.5, 3.0]), torch.ones(5)
    y = Int8Linear(w.to(DEV), t.to(DEV))(q.to(DEV), scale=s.to(DEV))
    _check(y, q.numpy(), s.numpy(), w, t, None, torch.float32)


@pytest.mark.parametrize("rows", [1, 40])
def test_strided_rows_and_weights(rows):
    from chessfly.int8 import Int8Linear
    wide = _x(rows, 301, 3)
    w, t, b = _weight(90, 205, 4)
    w_wide = torch.zeros(90, 211, dtype=torch.int8)
    w_wide[:, 3:208] = w
    lin = Int8Linear(w_wide.to(DEV)[:, 3:208], t.to(DEV), b.to(DEV))
    x = wide[:, 7:212]
    ref = O.quantize(x.numpy())
    _check(lin(wide.to(DEV)[:, 7:212]), *ref, w, t, b, torch.float32)
    _check(lin(x.t().contiguous().to(DEV).t()), *ref, w, t, b, torch.float32)   # columns apart: copied
    _check(lin(wide.half().to(DEV)[:, 7:212]), *O.quantize(x.half().float().numpy()), w, t, b, torch.float32)
    _check(lin(x[:1].to(DEV).expand(5, -1)), *O.quantize(x[:1].expand(5, -1).numpy()), w, t, b, torch.float32)


def test_no_rows():
    from chessfly.int8 import Int8Linear, quantize_rows
    w, t, b = _weight(9, 12, 4)
    assert Int8Linear(w.to(DEV), t.to(DEV))(torch.zeros(0, 12, device=DEV)).shape == (0, 9)
    q, s = quantize_rows(torch.zeros(0, 12, device=DEV))
    assert q.shape == (0, 12) and s.shape == (0,)


def test_from_float():
    from chessfly.int8 import Int8Linear
    g = torch.Generator().manual_seed(0)
    weight, bias, x = torch.randn(77, 150, generator=g), torch.randn(77, generator=g), _x(6, 150, 1)
    lin = Int8Linear.from_float(weight.to(DEV), bias.to(DEV))
    qw, t = O.quantize(weight.numpy())
    _check(lin(x.to(DEV)), *O.quantize(x.numpy()), torch.from_numpy(qw), torch.from_numpy(t), bias, torch.float32)


def test_outputs_are_the_same_for_every_batch_around_them():
    """Integer sums are exact: a row's outputs have the same bits whatever the batch, and whatever kernel it takes."""
    from chessfly.int8 import Int8Linear
    x = _x(700, 333, 8).to(DEV)
    w, t, b = _weight(1111, 333, 9)
    lin = Int8Linear(w.to(DEV), t.to(DEV), b.to(DEV))
    whole = lin(x)
    for rows in (1, 5, 16, 17, 33, 64, 100, 250, 600):
        assert torch.equal(lin(x[:rows]), whole[:rows]), rows


def test_offsets_past_32_bits():
    """Rows over 2^31 elements apart, and more outputs than that."""
    from chessfly.int8 import Int8Linear, quantize_rows
    w, t, b = _weight(17001, 70, 9)
    lin = Int8Linear(w.to(DEV), t.to(DEV), b.to(DEV))
    apart, x = 1_150_000_000, _x(3, 70, 3, torch.float16).to(DEV)
    far = torch.empty(2 * apart + 70, dtype=torch.float16, device=DEV).as_strided((3, 70), (apart, 1))
    far.copy_(x)
    assert torch.equal(lin(far), lin(x))
    assert all(torch.equal(a, b) for a, b in zip(quantize_rows(far), quantize_rows(x)))
    del far
    x = torch.randn(130_000, 70, device=DEV)
    y = lin(x, torch.float16)
    for part in (slice(0, 9), slice(126_300, 126_340), slice(129_900, 130_000)):
        assert torch.equal(y[part], lin(x[part], torch.float16))


def test_another_stream_and_a_graph():
    from chessfly.int8 import Int8Linear
    x = _x(64, 333, 8).to(DEV)
    w, t, b = _weight(200, 333, 9)
    lin = Int8Linear(w.to(DEV), t.to(DEV), b.to(DEV))
    ref = lin(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = lin(x)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, ref)
    for rows in (1, 64):
        inp = x[:rows].clone()
        lin(inp)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = lin(inp)
        for seed in range(3):
            inp.copy_(_x(rows, 333, 20 + seed))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, lin(inp)), (rows, seed)


def test_refusals():
    from chessfly.int8 import Int8Linear, quantize_rows
    w, t, b = _weight(9, 12, 4)
    w, t, b = w.to(DEV), t.to(DEV), b.to(DEV)
    lin = Int8Linear(w, t, b)
    x = torch.zeros(3, 12, device=DEV)
    for call in (lambda: Int8Linear(w.float(), t, b), lambda: Int8Linear(w, t[:5], b), lambda: Int8Linear(w, t, b.half()),
                 lambda: Int8Linear(w, t.cpu()), lambda: Int8Linear(w[0], t), lambda: lin(x[:, :5]), lambda: lin(x[0]),
                 lambda: lin(x.double()), lambda: lin(x, out_dtype=torch.int8), lambda: lin(x.to(torch.int8)),
                 lambda: lin(x, scale=torch.ones(3, device=DEV)), lambda: lin(x.cpu()),
                 lambda: lin(x.to(torch.int8), scale=torch.ones(2, device=DEV)), lambda: quantize_rows(x.double()),
                 lambda: quantize_rows(x[0])):
        with pytest.raises(RuntimeError):
            call()
