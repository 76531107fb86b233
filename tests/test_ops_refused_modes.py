"""Derivatives and traces that the operators do not take part in are refused where they are asked for: they would come out
as zeros, and as programs without the operators. The refusals come before any look at a device, so the CPU shows them."""

import pytest
import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from odc_amd import ops

CALLS = {
    "layer_norm": lambda x: ops.layer_norm(x, 8),
    "add_layer_norm": lambda x: ops.add_layer_norm(x, x, 8)[0],
    "LayerNorm": lambda x: ops.LayerNorm(8, elementwise_affine=False)(x),
    "squared_norm": lambda x: ops.squared_norm([x]),
    "adamw_step": lambda x: ops.adamw_step([x], [x], [x], [x], step=1, lr=1e-3),
    "adamw_step_8bit": lambda x: ops.adamw_step_8bit([x], [x], [x], [x], [x], [x], step=1, lr=1e-3, seed=1),
    "dequantize_blocks": lambda x: ops.dequantize_blocks(x, x),
}


@pytest.mark.parametrize("name", CALLS)
def test_traces(name):
    x = torch.randn(4, 8)
    with pytest.raises(NotImplementedError, match="traced"):
        make_fx(CALLS[name])(x)
    with pytest.raises(NotImplementedError, match="traced"):
        torch.jit.trace(CALLS[name], (x,), check_trace=False)
    with pytest.raises(TypeError, match="GPU"):  # and behind them all is as before
        CALLS[name](x)


@pytest.mark.parametrize("name", ["layer_norm", "add_layer_norm", "LayerNorm", "squared_norm"])
def test_tangents(name):
    x = torch.randn(4, 8)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            CALLS[name](dual)
        with pytest.raises(TypeError, match="GPU"):  # beside it tensors without a tangent are as before
            CALLS[name](x)
        with forward_ad._set_fwd_grad_enabled(False), pytest.raises(TypeError, match="GPU"):
            CALLS[name](dual)


@pytest.mark.parametrize("place", range(4))
def test_tangents_of_every_argument(place):
    tensors = [torch.randn(4, 8), torch.randn(4, 8), torch.ones(8), torch.ones(8)]
    with forward_ad.dual_level():
        tensors[place] = forward_ad.make_dual(tensors[place], torch.ones_like(tensors[place]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            ops.add_layer_norm(*tensors[:2], 8, *tensors[2:])
