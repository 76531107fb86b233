"""Operators of a training step around the gathers and scatter-accumulates, as hand-written HIP kernels for
MI355X (``include/odc_ops.h``):

* ``layer_norm`` / ``add_layer_norm`` and the ``LayerNorm`` module: forward and backward, with the reduction of the
  weight's and the bias's gradient, and the residual addition in front of the norm;
* ``adamw_step`` / ``adamw_step_8bit`` and the ``AdamW`` optimizer: one AdamW step over many tensors (the shards that
  ``pre_optimizer_step`` has handed their gradients), states in fp32 or in 8 bits, gradient clipping without a
  round trip to the host, the compute-dtype copy of the parameters written on the way;
* ``squared_norm`` of many tensors, ``dequantize_blocks`` to read states in 8 bits as values.

Everything is launched on the current stream of the tensors' device; the same inputs give the same bits. There is
no CPU path: tensors that are not on the GPU are refused.
"""

from odc_amd.ops.norm import LayerNorm, add_layer_norm, layer_norm
from odc_amd.ops.optim import AdamW, adamw_step, adamw_step_8bit, dequantize_blocks, squared_norm

__all__ = [
    "LayerNorm",
    "layer_norm",
    "add_layer_norm",
    "AdamW",
    "adamw_step",
    "adamw_step_8bit",
    "squared_norm",
    "dequantize_blocks",
]
