"""Layer norm, forward and backward."""

from __future__ import annotations

from typing import Optional, Sequence, Tuple, Union

import torch
from torch import Tensor

from odc_amd import _native

_host_path = _native.load_ops()


def layer_norm(input: Tensor, normalized_shape: Union[int, Sequence[int]], weight: Optional[Tensor] = None,
               bias: Optional[Tensor] = None, eps: float = 1e-5) -> Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimensions of ``input``, as
    ``torch.nn.functional.layer_norm`` outside of autocast: same arguments, same result up to rounding, differentiable once
    (a second derivative, a forward-mode one and a trace are refused).

    ``input`` is bf16, fp16 or fp32; ``weight`` and ``bias`` have its dtype or are fp32, and their gradients come in
    theirs. Rows may lie at any stride (slices of a wider tensor, expanded rows); what is not rows of neighbouring
    elements is copied first. ``torch.autocast`` changes nothing: torch's own runs in fp32 under it and returns fp32, this one
    returns the dtype of ``input`` (sums are fp32 in either). Statistics and sums are fp32; the reduction of the weight's gradient over the rows has
    a fixed order, so gradients are the same from run to run."""
    return _host_path.layer_norm(input, None, normalized_shape, weight, bias, eps)


def add_layer_norm(input: Tensor, residual: Tensor, normalized_shape: Union[int, Sequence[int]],
                   weight: Optional[Tensor] = None, bias: Optional[Tensor] = None, eps: float = 1e-5) -> Tuple[Tensor, Tensor]:
    """``total = input + residual; return layer_norm(total, ...), total`` in one pass: the residual addition of a
    pre-norm block. The two have one dtype (under autocast too: a bf16 branch is cast by the caller before it joins an fp32
    residual stream, or the stream kept in bf16). ``total`` has it, and it is what is normalised; in backward the gradient that
    comes back through ``total`` is added in the same pass."""
    return _host_path.layer_norm(input, residual, normalized_shape, weight, bias, eps)


class LayerNorm(torch.nn.LayerNorm):
    """``torch.nn.LayerNorm`` (same arguments, parameters and state dict) computed by ``layer_norm``, whatever autocast is
    set to; with a ``residual``, by ``add_layer_norm``."""

    def forward(self, input: Tensor, residual: Optional[Tensor] = None):
        return _host_path.layer_norm(input, residual, self.normalized_shape, self.weight, self.bias, self.eps)
