"""The AdamW step over many tensors, with states in fp32 or in 8 bits, and the norm that clips its gradients.

The formulas, in fp32 whatever the tensors' dtypes, with ``t = step``::

    g = grad * grad_scale * min(1, max_norm / (grad_scale * sqrt(squared_norm) + 1e-6))
    m = beta1 * m + (1 - beta1) * g
    v = beta2 * v + (1 - beta2) * g * g
    p = p * (1 - lr * weight_decay) - lr / (1 - beta1**t) * m / (sqrt(v) / sqrt(1 - beta2**t) + eps)

States in 8 bits. ``m`` and the root of ``v`` are e4m3 numbers (``torch.float8_e4m3fn``) that share a power of two
(``torch.float8_e8m0fnu``) in blocks of 32 neighbours: 8.25 bits per value, the block format that the hardware's
own scaled conversions use. The root spans the range of ``v`` in half the exponent, 17 binades of the root below a
block's largest value, 35 of ``v``. Codes lie 6 to 12 % apart, while an average with ``beta2 = 0.999`` moves by
0.1 % in a step: rounded to the nearest code it would never move. So a value between two codes becomes one of them by
a random number, such that its expectation is kept, that of ``m`` and that of ``v`` (the root's square). The numbers
are a function of ``seed``, the tensor's place in the list and the element's in the tensor: the same seed, the same
bits, another seed for every step. A ``v`` that is not zero is never stored as zero. This step's update is made from
``m`` and ``v`` as computed, before they are rounded.

Sums, products and the clipping factor are rounded to the nearest; the root of ``v`` and the reciprocal of the denominator are the
hardware's, within a unit of the last place each. In 8 bits that can make a code the other neighbour's where its random number is as
near to the share of the way, as any rounding can.
"""

from __future__ import annotations

import math
from typing import Optional, Sequence, Tuple

import torch
from torch import Tensor

from odc_amd import _native
from odc_amd.fsdp.shard_copies import shards_may_have_changed

_host_path = _native.load_ops()

BLOCK = 32  # elements of a state in 8 bits that share a scale


def squared_norm(tensors: Sequence[Tensor]) -> Tensor:
    """The sum of the squares of all elements of all tensors, as an fp32 scalar on their device: two launches for up
    to 320 tensors, no round trip to the host. Shards of one model: sum it over the ranks (``all_reduce``) before
    clipping by it. It has no derivative: where a tensor requires a gradient, a backward pass through the result raises."""
    if not isinstance(tensors, (list, tuple)):
        tensors = list(tensors)
    total = _host_path.squared_norm(tensors)
    if total is None:  # dtypes differ
        by_dtype = {}
        for t in tensors:
            by_dtype.setdefault(t.dtype, []).append(t)
        total = sum(_host_path.squared_norm(group) for group in by_dtype.values())
    return total


def adamw_step(params: Sequence[Tensor], grads: Sequence[Tensor], exp_avgs: Sequence[Tensor], exp_avg_sqs: Sequence[Tensor], *,
               step: int, lr: float, betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.0,
               grad_scale: float = 1.0, squared_norm: Optional[Tensor] = None, max_norm: Optional[float] = None,
               copies: Optional[Sequence[Tensor]] = None, seed: Optional[int] = None) -> None:
    """One AdamW step (see the module) over all tensors of the lists, in place, in one launch for up to 80 tensors (66 with
    copies; 57 and 50 with states in 8 bits).

    ``params`` are fp32 or bf16, ``grads`` fp32, bf16 or fp16, the states fp32; every list has one dtype, and the
    tensors of a place have one shape and layout, dense, at any alignment; what is written overlaps nothing else of the
    call. ``step`` counts from 1. ``squared_norm`` (a scalar on the device, see the function) and ``max_norm`` come
    together and clip the gradients; ``grad_scale`` multiplies them first (1 / W for sums over W ranks). A norm that is not
    finite is not looked at by the host: NaN makes every parameter NaN, as the formula says. ``copies`` (bf16 or fp16, of
    fp32 parameters) receive the new parameters. Parameters in bf16 are rounded to the nearest value, which loses updates
    of less than half a unit in their last place, or, where ``seed`` is given, by its random numbers."""
    _host_path.adamw(params, grads, exp_avgs, None, exp_avg_sqs, None, copies, _norm(squared_norm, max_norm), step, lr, *betas, eps,
                     weight_decay, grad_scale, 0.0 if max_norm is None else max_norm, seed)


def adamw_step_8bit(params: Sequence[Tensor], grads: Sequence[Tensor], exp_avgs: Sequence[Tensor], exp_avg_scales: Sequence[Tensor],
                    exp_avg_roots: Sequence[Tensor], exp_avg_root_scales: Sequence[Tensor], *, step: int, lr: float,
                    betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.0, grad_scale: float = 1.0,
                    squared_norm: Optional[Tensor] = None, max_norm: Optional[float] = None, copies: Optional[Sequence[Tensor]] = None,
                    seed: int) -> None:
    """``adamw_step`` with states in 8 bits: ``exp_avgs`` and ``exp_avg_roots`` hold a ``float8_e4m3fn`` code for
    every element (in the order of the parameter's memory), their scales a ``float8_e8m0fnu`` for every 32 of them.
    States to begin with are zeros, scales included (``torch.zeros(..., dtype=torch.uint8).view(dtype)``)."""
    _host_path.adamw(params, grads, exp_avgs, exp_avg_scales, exp_avg_roots, exp_avg_root_scales, copies, _norm(squared_norm, max_norm),
                     step, lr, *betas, eps, weight_decay, grad_scale, 0.0 if max_norm is None else max_norm, seed)


def _norm(squared_norm, max_norm):
    if (squared_norm is None) != (max_norm is None):
        raise ValueError("squared_norm and max_norm come together")
    return squared_norm


def dequantize_blocks(codes: Tensor, scales: Tensor, dtype: torch.dtype = torch.float32) -> Tensor:
    """What a state in 8 bits stands for: ``codes * scales``, 32 neighbouring codes to a scale, rounded once into ``dtype``. 4
    significant bits times a power of two, so it is exact in fp32 up to scales of 2^119, in bf16 with scales of 2^-124 to 2^119: all
    that the step writes lie there. Of a sharded parameter's states: what this rank has of them, as long as the
    largest shard needs (zeros behind its own)."""
    return _host_path.dequantize_blocks(_local(codes), _local(scales), dtype)


class AdamW(torch.optim.Optimizer):
    """AdamW over the fused steps above, for plain parameters and for the sharded ones of ``fully_shard`` and FSDP1.

    ``state_bits``: 32 (``exp_avg``, ``exp_avg_sq`` as in torch's AdamW) or 8 (``exp_avg``, ``exp_avg_root`` and their
    scales; 2.06 bytes per element instead of 8). ``max_norm`` clips the gradients by their norm over all parameters of
    the optimizer; where these are shards, give ``step`` the ``squared_norm`` summed over the ranks. ``seed`` sets
    the random roundings: of states in 8 bits, and of parameters in bf16 beside those or with ``stochastic_params``.

    States of a sharded parameter (a DTensor) are DTensors, so that torch's distributed checkpoint saves every rank's. In
    8 bits they are blocks of one shard's memory: one row for each shard, as long as the largest needs. They are read again for the
    same sharding; for another one their shapes do not match, and loading them raises.

    ``step`` may not be captured into a HIP graph: the step's number would be a constant of it."""

    def __init__(self, params, lr: float = 1e-3, betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, *, state_bits: int = 32, max_norm: Optional[float] = None, seed: int = 0,
                 stochastic_params: bool = False):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits is 8 or 32, not {state_bits}")
        if not (lr >= 0 and eps >= 0 and weight_decay >= 0):
            raise ValueError("lr, eps and weight_decay are not negative")
        if not all(0 <= b < 1 for b in betas):
            raise ValueError(f"betas lie in [0, 1): {betas}")
        if max_norm is not None and not max_norm >= 0:
            raise ValueError(f"max_norm is not negative: {max_norm}")
        self.state_bits, self.max_norm, self.seed, self.stochastic_params = state_bits, max_norm, int(seed), stochastic_params
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))

    def __getstate__(self):
        own = ("state_bits", "max_norm", "seed", "stochastic_params")
        return {**super().__getstate__(), **{name: getattr(self, name) for name in own}}

    @torch.no_grad()
    def step(self, closure=None, *, grad_scale: float = 1.0, squared_norm: Optional[Tensor] = None):
        """One step of every parameter that has a gradient. ``squared_norm``: see the class."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW.step cannot be captured into a graph: the step's number would be a constant of it")
        if squared_norm is not None and self.max_norm is None:
            raise ValueError("squared_norm without max_norm: there is nothing to clip to")
        calls, sharded, idle = {}, [], []
        for number, group in enumerate(self.param_groups):
            for p in group["params"]:
                grad = p.grad
                if grad is None:
                    continue
                param, grad = _local(p), _local(grad)
                if param is not p:
                    sharded.append(p)
                if grad.layout is not torch.strided:
                    raise TypeError("AdamW: sparse gradients are not supported")
                if not param.numel():
                    idle.append((p, param))
                    continue
                if not (grad.is_contiguous() and param.is_contiguous()) and grad.stride() != param.stride():
                    grad = torch.empty_like(param, dtype=grad.dtype).copy_(grad)
                state = self.state.get(p) or {}  # (reading self.state[p] would leave an empty one behind)
                key = (number, state["step"] + 1 if state else 1, param.device, param.dtype, grad.dtype)
                call = calls.get(key)
                if call is None:
                    call = calls[key] = ([], [], [], [])
                for place, value in zip(call, (p, param, grad, state)):
                    place.append(value)
        if squared_norm is None and self.max_norm is not None and calls:
            grads = [grad for _, _, grads, _ in calls.values() for grad in grads]
            # The norm of this rank's gradients is not that of all ranks'. (Where they are zero they are zero whatever they are clipped by:
            # torch's get_optimizer_state_dict begins the states by such a step.)
            shards = torch.distributed.is_available() and torch.distributed.is_initialized() and (
                any(p.device_mesh.size() > 1 for p in sharded if hasattr(p, "device_mesh"))
                or any(_is_flat_shard(p) for owners, _, _, _ in calls.values() for p in owners if hasattr(p, "_unpadded_unsharded_size")))
            if shards and any(bool(grad.any()) for grad in grads):
                raise ValueError("the parameters are shards: give step() the squared_norm of their gradients, summed over the ranks")
            squared_norm = _host_squared_norm(grads)
        # Every call is checked before the first is made: a step that is refused has written nothing.
        prepared, begun = [], []
        try:
            for place, ((number, step, device, _, _), (owners, params, grads, states)) in enumerate(calls.items()):
                group = self.param_groups[number]
                # another seed for every step, and for every call of a step
                seed = (self.seed * 0x9E3779B1 + step * 0x85EB + place * 0x27D4EB2F) & 0xFFFFFFFF
                if step == 1:
                    for p, param, state in zip(owners, params, states):
                        if not state:
                            begun.append(p)
                            self._begin(state, p, param)
                            self.state[p] = state
                if self.state_bits == 8:
                    lists = [[s[name] for s in states] for name in _STATES_8BIT]
                    if sharded:
                        lists = [[_first(t, param.numel(), per) for t, param in zip(one, params)] for one, per in zip(lists, (1, BLOCK) * 2)]
                else:
                    exp_avgs, exp_avg_sqs = ([_local(s[name]) for s in states] for name in ("exp_avg", "exp_avg_sq"))
                    lists, seed = (exp_avgs, None, exp_avg_sqs, None), seed if self.stochastic_params else None
                prepared.append((step, states, _host_path.adamw_prepare(
                    params, grads, *lists, None, None if squared_norm is None else squared_norm.to(device), step, float(group["lr"]),
                    *group["betas"], group["eps"], group["weight_decay"], grad_scale, 0.0 if self.max_norm is None else self.max_norm, seed)))
            for p, param in idle:  # nothing to step, but a shard without elements has states as the other ranks' have
                if not self.state.get(p):
                    begun.append(p)
                    self._begin(self.state[p], p, param)
        except BaseException:
            for p in begun:
                self.state.pop(p, None)
            raise
        try:
            for step, states, call in prepared:
                _host_path.adamw_launch(call)
                for state in states:
                    state["step"] = step
            for p, _ in idle:
                self.state[p]["step"] += 1
        finally:  # (a launch that fails leaves the ones in front of it done)
            if sharded:
                torch.autograd.graph.increment_version(sharded)  # of a DTensor: its local tensor has a counter of its own
            shards_may_have_changed()
        return loss

    def _begin(self, state, p, param):
        state["step"] = 0
        if self.state_bits == 32:
            state["exp_avg"] = torch.zeros_like(p, dtype=torch.float32, memory_format=torch.preserve_format)
            state["exp_avg_sq"] = torch.zeros_like(p, dtype=torch.float32, memory_format=torch.preserve_format)
            return
        n, dtypes = param.numel(), (torch.float8_e4m3fn, torch.float8_e8m0fnu) * 2
        shards = None
        if hasattr(p, "placements"):
            n, shards = _shards_of(p, n)
        for name, size, dtype in zip(_STATES_8BIT, (n, -(-n // BLOCK)) * 2, dtypes):
            value = torch.zeros(size, dtype=torch.uint8, device=param.device).view(dtype)
            state[name] = value if shards is None else _one_of(value, p, shards)

    def load_state_dict(self, state_dict):
        """As ``torch.optim.Optimizer.load_state_dict``, which takes every state for one of its parameter's dtype:
        here they keep their own. In 32 bits the states of ``torch.optim.AdamW`` are read too (the step's number, a tensor
        there, becomes an int); options of its that change the step, and that this one does not have, are refused."""
        saved = [i for g in state_dict["param_groups"] for i in g["params"]]
        names = set(_STATES_8BIT if self.state_bits == 8 else ("exp_avg", "exp_avg_sq")) | {"step"}
        for state in state_dict["state"].values():
            if state and set(state) != names:
                raise ValueError(f"the states are those of another optimizer: {sorted(state)}, not {sorted(names)} (state_bits={self.state_bits})")
        for group in state_dict["param_groups"]:
            coupled = group.get("weight_decay") and group.get("decoupled_weight_decay") is False  # torch.optim.Adam's
            for name, wrong in (("amsgrad", group.get("amsgrad")), ("maximize", group.get("maximize")), ("decoupled_weight_decay=False", coupled)):
                if wrong:
                    raise ValueError(f"the states are those of another optimizer: {name} is not supported")
        super().load_state_dict(state_dict)
        for i, p in zip(saved, (p for g in self.param_groups for p in g["params"])):
            for name, value in state_dict["state"].get(i, {}).items():
                if name == "step":
                    self.state[p][name] = int(value)
                elif isinstance(value, Tensor):
                    self.state[p][name] = value.detach().clone().to(p.device)


_STATES_8BIT = ("exp_avg", "exp_avg_scale", "exp_avg_root", "exp_avg_root_scale")
_PLAIN = (Tensor, torch.nn.Parameter)
_host_squared_norm = squared_norm


def _shards_of(p, n: int) -> Tuple[int, Tuple[int, ...]]:
    """Elements of the largest shard of a DTensor (``n`` of them are here), and into how many it is split along each of
    its dimensions."""
    longest, shards = list(p.shape), [1] * p.dim()
    for k, placement in enumerate(p.placements):
        dim = getattr(placement, "dim", None)
        if dim is not None:
            longest[dim], shards[dim] = -(-longest[dim] // p.device_mesh.size(k)), shards[dim] * p.device_mesh.size(k)
    return max(n, math.prod(longest)), tuple(shards)


def _one_of(value: Tensor, p, shards: Tuple[int, ...]) -> Tensor:
    """``value`` as the part of this rank of a DTensor that is placed as ``p`` is: one row for each of the shards."""
    from torch.distributed.tensor import DTensor

    shape = (*shards, value.numel())
    stride = [math.prod(shape[k + 1:]) for k in range(len(shape))]
    return DTensor.from_local(value.view(*(1 for _ in shards), -1), p.device_mesh, p.placements, run_check=False, shape=torch.Size(shape),
                              stride=tuple(stride))


def _first(state: Tensor, elems: int, per: int) -> Tensor:
    """Of a state (of a DTensor: its part here, which is as long as the largest shard needs) what belongs to ``elems``
    elements."""
    local, n = _local(state), -(-elems // per)
    return local if local is state or local.numel() == n else local.view(-1)[:n]


def _is_flat_shard(p: Tensor) -> bool:
    """Whether ``p`` is FSDP1's flat parameter of a model whose other parts are on other ranks. (With ``use_orig_params``
    the parameters are plain tensors, and nothing says that they are shards.)"""
    return p.numel() < p._unpadded_unsharded_size.numel()


def _local(t: Tensor) -> Tensor:
    """The memory behind a parameter, a gradient or a state: of a DTensor its shard here."""
    return t if type(t) in _PLAIN else getattr(t, "_local_tensor", t)
