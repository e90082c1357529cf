"""GPU tests of clipping by the norm of all gradients, against float64."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from oracle import readout as O
from oracle.operators import TINY, UNIT

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


def params(shapes, types, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    out = []
    for i, s in enumerate(shapes):
        t = TYPES[types[i % len(types)]]
        p = torch.nn.Parameter(torch.zeros(s, dtype=t, device=DEV))
        p.grad = (torch.randn(s, generator=g) * scale * 10.0 ** -(i % 4)).to(t).to(DEV)
        out.append(p)
    return out


def check(ps, limit, norm_type=2.0):
    """The norm is summed in float64 and rounded once.  The factor has the limit's, the sum's and the quotient's roundings besides
    the norm's, and each product one to float32 and one to its type."""
    from chessfly.clip import clip_grad_norm_
    before = [p.grad.double().cpu().numpy() for p in ps]
    versions = [p.grad._version for p in ps]
    norm = clip_grad_norm_(ps, limit, norm_type)
    want, scaled = O.clip(before, limit, norm_type)
    assert norm.dtype == torch.float32 and norm.shape == () and norm.device.type == "cuda"
    assert abs(float(norm) - want) <= 2.0 ** -23 * want
    for p, b, e, was in zip(ps, before, scaled, versions):
        t = str(p.dtype)[6:]
        got = p.grad.double().cpu().numpy()
        assert p.grad._version > was
        if limit / (want + 1e-6) >= 1 + 1e-5:
            assert np.array_equal(got, b)
        else:
            assert (np.abs(got - e) <= 1.01 * ((6 * 2.0 ** -24 + UNIT[t]) * np.abs(e) + TINY[t])).all()


SETS = {
    "one element": [(1,)], "one tensor": [(1000,)], "a chunk and its neighbours": [(8191,), (8192,), (8193,), (16383,), (16385,)],
    "odd": [(3, 5), (7,), (1, 1, 1), (33, 65), (129,)], "empty ones": [(0,), (4, 0), (17,), (0, 3)], "none but empty": [(0,)],
    "large": [(3000, 2333), (10,), (4168, 700)], "as many as a launch holds": [(i + 1,) for i in range(128)],
    "one more": [(i + 1,) for i in range(129)], "many": [(17 * i % 4001,) for i in range(700)],
}


@pytest.mark.parametrize("norm_type", [2.0, math.inf])
@pytest.mark.parametrize("limit", [0.1, 1e6])
@pytest.mark.parametrize("types", [["float32"], ["float16"], ["bfloat16"], list(TYPES)])
@pytest.mark.parametrize("name", list(SETS))
def test_sets(name, types, limit, norm_type):
    check(params(SETS[name], types, seed=len(name)), limit, norm_type)


def test_more_sums_than_a_workgroup_adds():
    """Launches of 128 large tensors each: a join between the passes."""
    ps = params([(600_000,)] * 260, ["float32"], seed=3)
    check(ps, 0.5)


def test_sums_of_squares_beyond_float32():
    for size in (1e25, 1e-25):
        check(params([(100_000,), (5,)], ["float32"], scale=size), 0.25 * size)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("norm_type", [2.0, math.inf])
def test_gradients_that_are_not_finite(bad, norm_type):
    """As torch's: a NaN norm makes all NaN, an infinite one all zero but what was infinite."""
    from chessfly.clip import clip_grad_norm_, grad_norm
    ours, theirs = (params([(5000,), (70,)], ["float32"]) for _ in range(2))
    for ps in (ours, theirs):
        ps[0].grad[4321] = bad
    before = [p.grad.clone() for p in ours]
    with pytest.raises(RuntimeError, match="norm is"):
        clip_grad_norm_(ours, 1.0, norm_type, error_if_nonfinite=True)
    assert all(torch.equal(p.grad.nan_to_num(7), b.nan_to_num(7)) for p, b in zip(ours, before))
    n = clip_grad_norm_(ours, 1.0, norm_type)
    m = torch.nn.utils.clip_grad_norm_(theirs, 1.0, norm_type)
    assert torch.equal(n.nan_to_num(7), m.nan_to_num(7))
    for p, q in zip(ours, theirs):
        assert torch.equal(p.grad.nan_to_num(7), q.grad.nan_to_num(7)) and torch.equal(p.grad.isnan(), q.grad.isnan())


def test_layouts():
    """Transposed, permuted, at odd addresses, of parts of larger tensors: what lies between stays."""
    base = torch.randn(5000, device=DEV, dtype=torch.bfloat16)
    large = torch.randn(40, 50, device=DEV)
    ps = [torch.nn.Parameter(torch.zeros(s, device=DEV, dtype=t)) for s, t in
          [((30, 20), torch.float32), ((2, 3, 4, 5), torch.float32), ((4097,), torch.bfloat16), ((20, 25), torch.float32)]]
    ps[0].grad = torch.randn(20, 30, device=DEV).t()
    ps[1].grad = torch.randn(2, 4, 5, 3, device=DEV).permute(0, 3, 1, 2)
    ps[2].grad = base[3:4100]
    ps[3].grad = large[5:25, 10:35]
    ends, rest = base.clone(), large.clone()
    check(ps, 0.5)
    assert torch.equal(base[:3], ends[:3]) and torch.equal(base[4100:], ends[4100:])
    rest[5:25, 10:35] = large[5:25, 10:35]
    assert torch.equal(large, rest)


def test_single_tensors_none_and_the_norm_alone():
    from chessfly.clip import clip_grad_norm_, grad_norm
    p = params([(1000,)], ["float32"])[0]
    before = p.grad.clone()
    n = grad_norm(p)
    assert torch.equal(p.grad, before) and torch.equal(n, grad_norm([p, torch.nn.Parameter(torch.zeros(3, device=DEV))]))
    assert torch.equal(n, clip_grad_norm_((q for q in [p]), 1e9)) and torch.equal(p.grad, before)
    assert torch.equal(grad_norm([p, p]), torch.tensor(O.clip([before.cpu().numpy()] * 2, 1.0)[0], dtype=torch.float32, device=DEV))
    assert float(grad_norm(p, math.inf)) == float(before.abs().max())
    clip_grad_norm_(p, 0.0)
    assert not p.grad.any()


def test_refuses():
    from chessfly.clip import clip_grad_norm_
    a, b = params([(8, 8), (8, 8)], ["float32"])
    before = a.grad.clone()
    for bad in ([a, a], [a, b]):
        b.grad = a.grad if bad[1] is b else b.grad
        with pytest.raises(RuntimeError, match="overlap"):
            clip_grad_norm_(bad, 1.0)
    shared = torch.zeros(100, device=DEV)
    a.grad, b.grad = shared[:64].view(8, 8), shared[36:].view(8, 8)
    with pytest.raises(RuntimeError, match="overlap"):
        clip_grad_norm_([a, b], 1.0)
    for grad in (torch.ones(1, 8, device=DEV).expand(8, 8), torch.ones(20, device=DEV).as_strided((8, 8), (1, 1))):
        a.grad = grad
        with pytest.raises(RuntimeError, match="overlap"):
            clip_grad_norm_(a, 1.0)
    with pytest.raises(RuntimeError, match="norm_type"):
        clip_grad_norm_(b, 1.0, 3.0)
    with pytest.raises(RuntimeError, match="max_norm"):
        clip_grad_norm_(b, float("nan"))
    d = torch.nn.Parameter(torch.zeros(4, device=DEV, dtype=torch.float64))
    d.grad = torch.ones_like(d)
    with pytest.raises(RuntimeError, match="float32"):
        clip_grad_norm_(d, 1.0)
    assert before.isfinite().all()


def test_in_a_graph_and_on_streams():
    from chessfly.clip import clip_grad_norm_
    ps = params(SETS["odd"] + [(200_000,)], list(TYPES))
    graph = torch.cuda.CUDAGraph()
    clip_grad_norm_(ps, 1.0)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        norm = clip_grad_norm_(ps, 1.0)
    for seed in range(4):
        fresh = [torch.randn(p.shape, generator=torch.Generator().manual_seed(seed)).to(p.dtype).to(DEV) for p in ps]
        for p, f in zip(ps, fresh):
            p.grad.copy_(f)
        graph.replay()
        torch.cuda.synchronize()
        got = [p.grad.clone() for p in ps]
        for p, f in zip(ps, fresh):
            p.grad.copy_(f)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            again = clip_grad_norm_(ps, 1.0)
        torch.cuda.synchronize()
        assert torch.equal(norm, again) and all(torch.equal(g, p.grad) for g, p in zip(got, ps))
