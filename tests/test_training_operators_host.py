"""CPU tests of the read-out loss's and the clipping's entry points: what their host side refuses, before any launch."""

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


def _loss(lib, **kw):
    return lib.fly_readout_loss(*{**dict(
        x=P, type=0, ldx=8, rows=4, d=8, w=P, ldw=8, v=9, bias=P, bias_type=0, legal=None, ldl=0, index=P, index_type=4,
        weight=None, k=1, loss=P, row_scale=None, grad_scale=1.0, gx=P, ldgx=8, gw=P, ldgw=8, gb=P, ws=P, ws_bytes=0,
        stream=None), **kw}.values())


def test_readout_loss_refuses(lib):
    for null in ("x", "w", "index"):
        _refused(_loss(lib, **{null: None}), lib, b"null")
    for ld in ("ldx", "ldw", "ldgx", "ldgw"):
        _refused(_loss(lib, **{ld: 7}), lib, b"overlap")
    _refused(_loss(lib, legal=P, ldl=8), lib, b"overlap")
    for size in (dict(rows=-1), dict(rows=1 << 40), dict(d=0), dict(d=(1 << 16) + 1), dict(v=0), dict(v=(1 << 20) + 1)):
        _refused(_loss(lib, **size), lib, b"range")
    for t in (-1, 3):
        _refused(_loss(lib, type=t), lib, b"float32")
        _refused(_loss(lib, bias_type=t), lib, b"bias")
    _refused(_loss(lib, index_type=0), lib, b"int32")
    _refused(_loss(lib, k=0), lib, b"k must")
    _refused(_loss(lib, k=1025), lib, b"k must")
    _refused(_loss(lib, loss=None, gx=None, gw=None, gb=None), lib, b"neither")
    _refused(_loss(lib), lib, b"workspace")
    _refused(_loss(lib, ws=P + 8, ws_bytes=1 << 40), lib, b"workspace")


def test_readout_workspace(lib):
    need = lambda *a: lib.fly_readout_loss_workspace(*a)
    assert need(0, 0, 8, 9, 1, 7) == 0
    assert need(0, -1, 8, 9, 1, 7) == 0 and need(5, 4, 8, 9, 1, 7) == 0 and need(0, 4, 8, 9, 0, 7) == 0
    assert 0 < need(1, 4, 8, 9, 1, 0) < need(1, 4, 8, 9, 1, 7)
    # rows beyond a piece take no more: the logits are not kept
    assert need(2, 1 << 22, 64, 32000, 1, 7) == need(2, 1 << 30, 64, 32000, 1, 7) < (9 << 30) // 2


def _clip(lib, grads=(P,), sizes=(4,), types=(0,), kind=2, limit=1.0, norm=P, ws=P, need=1 << 20):
    n = len(sizes)
    arr = lambda t, v: (t * max(n, 1))(*v)
    return lib.fly_clip_gradients(arr(ctypes.c_void_p, grads), arr(ctypes.c_int64, sizes), arr(ctypes.c_int32, types), n, kind,
                                  limit, norm, ws, need, None)


def test_clip_refuses(lib):
    _refused(_clip(lib, sizes=(-1,)), lib, b"size")
    _refused(_clip(lib, types=(3,)), lib, b"float32")
    _refused(_clip(lib, kind=1), lib, b"norm")
    _refused(_clip(lib, limit=float("nan")), lib, b"limit")
    _refused(_clip(lib, norm=None), lib, b"null")
    _refused(_clip(lib, grads=(None,)), lib, b"null")
    _refused(_clip(lib, grads=(P + 2,)), lib, b"misaligned")
    _refused(_clip(lib, need=0), lib, b"workspace")
    _refused(_clip(lib, ws=P + 4), lib, b"workspace")
    _refused(_clip(lib, grads=(P, P), sizes=(4, 4), types=(0, 0)), lib, b"overlap")
    _refused(_clip(lib, grads=(P + 12, P), sizes=(4, 4), types=(0, 0)), lib, b"overlap")


def test_clip_workspace(lib):
    need = lambda sizes: lib.fly_clip_workspace((ctypes.c_int64 * len(sizes))(*sizes), (ctypes.c_int32 * len(sizes))(), len(sizes))
    assert need([]) == 8 and need([0]) == 8 and need([1]) == 16
    assert need([1 << 34]) == 8 * 2049


def test_operators_refuse_cpu_tensors():
    from chessfly.clip import clip_grad_norm_, grad_norm
    from chessfly.readout import readout_loss, readout_loss_and_grad
    p = torch.nn.Parameter(torch.zeros(3))
    p.grad = torch.zeros(3)
    x, w, t = torch.zeros(2, 3), torch.zeros(4, 3), torch.zeros(2, dtype=torch.int64)
    for call in (lambda: clip_grad_norm_([p], 1.0), lambda: grad_norm(p), lambda: readout_loss(x, w, None, t),
                 lambda: readout_loss_and_grad(x, w, None, t)):
        with pytest.raises(RuntimeError, match="HIP device"):
            call()
    with pytest.raises(RuntimeError, match="max_norm"):
        clip_grad_norm_([p], -1.0)
    with pytest.raises(RuntimeError, match="reduction"):
        readout_loss(x, w, None, t, reduction="max")
    assert clip_grad_norm_([torch.nn.Parameter(torch.zeros(3))], 1.0) == 0
