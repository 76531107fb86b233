"""An eps that fp32 holds as a subnormal number, or as zero though it is none, is refused: the step's reciprocal takes such a
denominator for zero, and parameters that had no gradient yet became NaN."""

import ctypes

import pytest
import torch

from odc_amd import _native, ops


class Item(ctypes.Structure):
    """``odc_adamw_item`` of include/odc_ops.h."""

    _fields_ = [(n, ctypes.c_void_p) for n in ("param", "grad", "exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale", "copy")] + [("elems", ctypes.c_uint64)]


class Numbers(ctypes.Structure):
    """``odc_adamw_numbers``."""

    _fields_ = ([(n, ctypes.c_double) for n in ("lr", "beta1", "beta2", "eps", "weight_decay", "grad_scale", "max_norm")]
                + [("squared_norm", ctypes.c_void_p), ("step", ctypes.c_uint64), ("seed", ctypes.c_uint32)]
                + [(n, ctypes.c_int32) for n in ("stochastic", "param_dtype", "grad_dtype", "copy_dtype", "state_bits")])


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("eps,fine", [(0.0, True), (1.1754943508222875e-38, True), (1e-30, True), (1e-8, True),
                                      (1.17549e-38, False), (1e-40, False), (1e-46, False), (5e-324, False)])
def test_eps(eps, fine, bits):
    _native.load_ops()
    item = Item(*(0x1000 * (k + 1) for k in range(6)), None, 10)  # (nothing reads through them: the check launches nothing)
    numbers = Numbers(1e-3, 0.9, 0.999, eps, 0.0, 1.0, 0.0, None, 1, 0, 0, 2, 2, -1, bits)
    status = _native._ops_lib.odc_adamw_check(ctypes.byref(item), 1, ctypes.byref(numbers))
    assert (status == 0) == fine
    assert fine or b"eps" in _native._ops_lib.odc_ops_last_error()


@pytest.mark.gpu
def test_parameters_without_a_gradient_stay_numbers():
    p, g, m, v = (torch.full((40,), float(k), device="cuda") for k in (1, 0, 0, 0))
    with pytest.raises(RuntimeError, match="eps"):
        ops.adamw_step([p], [g], [m], [v], step=1, lr=0.1, eps=1e-40)
    ops.adamw_step([p], [g], [m], [v], step=1, lr=0.1, eps=1.2e-38)
    assert bool((p == 1).all())
