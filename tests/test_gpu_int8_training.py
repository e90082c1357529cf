"""GPU test of a network with an 8-bit read-out in training: the read-out is the float one."""

from __future__ import annotations

import copy

import pytest
import torch

from test_gpu_int8_head import DEV, _net

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("grad", [True, False])
def test_training_takes_the_float_read_out(grad):
    from chessfly.synthetic import synthetic_boards
    net = _net(torch.float32)
    x = torch.as_tensor(synthetic_boards(5, seed=3), device=DEV)
    with torch.no_grad():
        net.head_dtype = torch.int8
        rounded = net(x)[0]                        # what an 8-bit read-out gives
        net.head_dtype = torch.float32
        off = float((rounded - net(x)[0]).abs().max())
    net.train()
    state = copy.deepcopy(net.state_dict())
    out = {}
    for dtype in (torch.float32, torch.int8):
        net.load_state_dict(state)
        net.head_dtype = dtype
        with torch.set_grad_enabled(grad):
            out[dtype] = net(x)
        assert out[dtype][0].requires_grad == grad
    for a, b in zip(out[torch.float32], out[torch.int8]):
        assert float((a - b).detach().abs().max()) < 1e-3 * off
