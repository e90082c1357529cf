"""GPU tests at the ends of what the 8-bit and distillation entry points accept."""

from __future__ import annotations

import threading

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
ROWS = (1 << 26) + 5        # 64 threads for each row are 2^32, more than a launch holds
PARTS = [(i, min(i + (1 << 24) + 3, ROWS)) for i in range(0, ROWS, (1 << 24) + 3)]


def _rows(cols, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(ROWS, cols, generator=g, device=DEV, dtype=torch.float16)


def test_more_rows_than_a_launch_holds_to_8_bits():
    from chessfly.int8 import quantize_rows
    x = _rows(1, 1)
    whole = quantize_rows(x)
    for a, b in PARTS:
        assert all(torch.equal(w[a:b], p) for w, p in zip(whole, quantize_rows(x[a:b])))


def test_more_rows_than_a_launch_holds_of_logits():
    from chessfly.distill import TopLogits, distill_loss_and_grad, top_logits
    z = _rows(2, 1)
    legal = torch.rand(ROWS, 2, device=DEV) < 0.9
    lists = top_logits(_rows(2, 2), 1, 2.0, legal)
    scale = torch.rand(ROWS, device=DEV)
    whole = distill_loss_and_grad(z, lists, 2.0, legal, row_scale=scale)
    for a, b in PARTS:
        assert all(torch.equal(w[a:b], p) for w, p in zip(lists, top_logits(_rows(2, 2)[a:b], 1, 2.0, legal[a:b])))
        part = distill_loss_and_grad(z[a:b], TopLogits(*(t[a:b] for t in lists)), 2.0, legal[a:b], row_scale=scale[a:b])
        assert all(torch.equal(w[a:b], p) for w, p in zip(whole, part))


def _linear(k, seed):
    from chessfly.int8 import Int8Linear
    g = torch.Generator().manual_seed(seed)
    lin = Int8Linear.from_float(torch.randn(100, k, generator=g).to(DEV))
    x = torch.randn(32, k, generator=g).to(DEV)
    return lambda: lin(x), x


def _distill(cols, seed):
    from chessfly.distill import distill_loss_and_grad, top_logits
    g = torch.Generator().manual_seed(seed)
    z, lists = torch.randn(2, cols, generator=g).to(DEV), top_logits(torch.randn(2, cols, generator=g).to(DEV), 20)
    return lambda: torch.cat([t.flatten() for t in distill_loss_and_grad(z, lists)]), z


@pytest.mark.parametrize("k", [1000, 1030, 1500, 1550, 2000, 3000, 3072])
@pytest.mark.parametrize("rows", [9, 16, 17, 32])
def test_few_rows_of_every_size_in_lds(k, rows):
    """Rows alone and in a batch that another kernel takes have the same bits."""
    from chessfly.int8 import Int8Linear
    g = torch.Generator().manual_seed(k)
    lin = Int8Linear.from_float(torch.randn(100, k, generator=g).to(DEV))
    x = torch.randn(40, k, generator=g).to(DEV)
    assert torch.equal(lin(x[:rows]), lin(x)[:rows])


@pytest.mark.parametrize("make,large,small", [(_linear, 3050, 1100), (_distill, 1 << 20, 500_000)])
def test_large_and_small_calls_of_two_threads(make, large, small):
    """Calls that take much LDS and less of it, of one kernel, side by side."""
    calls = [make(large, 1)[0], make(small, 2)[0]]
    want, wrong = [c() for c in calls], []
    torch.cuda.synchronize()

    def work(call, ref):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(200):
                    if not torch.equal(call(), ref):
                        wrong.append("result")
        except Exception as e:   # a refused launch
            wrong.append(e)

    threads = [threading.Thread(target=work, args=a) for a in zip(calls, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong[:3]


@pytest.mark.parametrize("make,size", [(_linear, 3040), (_distill, 1 << 20), (_distill, 600_000)])
def test_calls_that_take_much_lds_in_a_graph(make, size):
    call, inp = make(size, 3)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for seed in range(3):
        g = torch.Generator().manual_seed(10 + seed)
        inp.copy_(torch.randn(inp.shape, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, call()), seed
