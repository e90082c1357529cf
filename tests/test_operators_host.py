"""CPU tests of the 8-bit and distillation entry points: what their host side refuses, before any launch."""

from __future__ import annotations

import ctypes

import pytest
import torch

from chessfly import _hip

P = 256    # a non-null, aligned address that no refused call reads


@pytest.fixture(scope="module")
def lib():
    return _hip.load()


def _refused(status: int, lib, word: bytes):
    assert status == 1 and word in lib.fly_last_error(), (status, lib.fly_last_error())


def test_quantize_rows_refuses(lib):
    call = lambda **kw: lib.fly_quantize_rows(*{**dict(x=P, x_type=0, ldx=8, rows=4, cols=8, q=P, ldq=8, scale=P,
                                                       stream=None), **kw}.values())
    _refused(call(x=None), lib, b"null")
    _refused(call(scale=None), lib, b"null")
    _refused(call(ldx=7), lib, b"size")
    _refused(call(ldq=7), lib, b"size")
    _refused(call(rows=-1), lib, b"size")
    _refused(call(x_type=3), lib, b"float32")


def test_int8_create_refuses(lib):
    out = ctypes.c_void_p()
    call = lambda **kw: lib.fly_int8_create(*{**dict(w=P, ldw=8, scale=P, bias=None, n=4, k=8, stream=None,
                                                     out=ctypes.byref(out)), **kw}.values())
    _refused(call(w=None), lib, b"null")
    _refused(call(scale=None), lib, b"null")
    _refused(call(n=0), lib, b"size")
    _refused(call(k=1 << 17, ldw=1 << 17), lib, b"size")
    _refused(call(ldw=7), lib, b"size")
    _refused(call(out=None), lib, b"out")
    assert lib.fly_int8_workspace(None, 0, 4) == 0
    assert lib.fly_int8_linear(None, P, 0, 8, None, 1, P, 0, 8, P, 1 << 20, None) == 1


def _top(lib, **kw):
    return lib.fly_top_logits(*{**dict(z=P, type=0, ldz=9, rows=2, cols=9, legal=None, ldl=0, k=3, temperature=1.0, values=P,
                                       index=P, tail=None, stream=None), **kw}.values())


def _distill(lib, **kw):
    return lib.fly_distill(*{**dict(z=P, type=0, ldz=9, rows=2, cols=9, legal=None, ldl=0, values=P, index=P, tail=None, k=3,
                                    temperature=1.0, loss=P, grad=P, ldg=9, row_scale=None, grad_scale=1.0,
                                    stream=None), **kw}.values())


@pytest.mark.parametrize("call", [_top, _distill])
def test_logits_refuses(lib, call):
    _refused(call(lib, z=None), lib, b"null")
    _refused(call(lib, ldz=8), lib, b"overlap")
    _refused(call(lib, cols=0), lib, b"range")
    _refused(call(lib, cols=(1 << 20) + 1, ldz=1 << 21), lib, b"range")
    _refused(call(lib, rows=-1), lib, b"range")
    _refused(call(lib, k=0), lib, b"k must")
    _refused(call(lib, k=257), lib, b"k must")
    for t in (0.0, -1.0, float("nan"), float("inf"), 1e-40):
        _refused(call(lib, temperature=t), lib, b"temperature")
    _refused(call(lib, legal=P, ldl=8), lib, b"mask")
    _refused(call(lib, type=3), lib, b"float32")
    _refused(call(lib, values=None), lib, b"values")
    _refused(call(lib, index=None), lib, b"index")


def test_distill_refuses(lib):
    _refused(_distill(lib, loss=None, grad=None), lib, b"neither")
    _refused(_distill(lib, ldg=8), lib, b"overlap")


def test_products_refuse_cpu_tensors():
    from chessfly.distill import TopLogits, distill_loss, distill_loss_and_grad, top_logits
    from chessfly.int8 import Int8Linear, quantize_rows
    z = torch.zeros(2, 9)
    teacher = TopLogits(torch.zeros(2, 3), torch.zeros(2, 3, dtype=torch.int32))
    for call in (lambda: quantize_rows(z), lambda: Int8Linear(z.to(torch.int8), torch.ones(2)),
                 lambda: top_logits(z, 3), lambda: distill_loss(z, teacher), lambda: distill_loss_and_grad(z, teacher)):
        with pytest.raises(RuntimeError, match="HIP device"):
            call()
