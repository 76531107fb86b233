"""A launch of odc_amd.ops is judged by its own status: what an earlier HIP call of the same thread failed with is
none of it."""

import ctypes
import re
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture
def hip():
    """torch's HIP runtime, the one that this process has loaded."""
    torch.cuda.init()
    paths = set(re.findall(r"/\S*libamdhip64\.so\S*", Path("/proc/self/maps").read_text()))
    assert len(paths) == 1, paths
    runtime = ctypes.CDLL(paths.pop())
    yield runtime
    runtime.hipGetLastError()


def leave_an_error(hip):
    """A question to the host about a device that is not there: it fails, and nothing else happens."""
    answer = ctypes.c_int()
    code = hip.hipDeviceGetAttribute(ctypes.byref(answer), 0, 9999)
    assert code != 0 and hip.hipPeekAtLastError() == code


class NormBackward(ctypes.Structure):
    """``odc_norm_backward`` of include/odc_ops.h."""

    _fields_ = ([(name, ctypes.c_void_p) for name in ("grad_output", "grad_total", "normalised", "weight", "mean", "rstd", "grad_input",
                                                      "grad_weight", "grad_bias", "workspace")]
                + [(name, ctypes.c_uint64) for name in ("workspace_bytes", "rows", "width", "grad_output_stride", "grad_total_stride",
                                                        "normalised_stride")]
                + [("dtype", ctypes.c_int32), ("weight_dtype", ctypes.c_int32)])


def test_an_earlier_error_is_no_launch_of_ours(hip):
    from odc_amd import _native, ops

    lib = _native._ops_lib
    gen = torch.Generator(device="cuda").manual_seed(0)

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    starts, gs = [randn(37 + k) for k in range(170)], [randn(37 + k) for k in range(170)]  # three launches of 80, 80 and 10
    codes = torch.arange(64, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    scales = torch.full((2,), 127, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu)
    shapes = [(5000, 96), (9, 20001), (3, 64)]  # in registers, wide, in one launch
    rows = [randn(*shape) for shape in shapes]
    grads = [randn(*shape) for shape in shapes]

    def backward(x, dy, out):
        """By the C ABI: autograd would make the call on a thread of its own."""
        mean, rstd = x.mean(1), torch.rsqrt(x.var(1, unbiased=False) + 1e-5)
        n, width = x.shape
        lib.odc_layer_norm_backward_workspace.argtypes = [ctypes.c_uint64, ctypes.c_uint64, ctypes.c_int32]
        workspace = torch.empty(lib.odc_layer_norm_backward_workspace(n, width, 2), dtype=torch.uint8, device="cuda")
        pointers = (dy, None, x, None, mean, rstd, *out, workspace)
        call = NormBackward(*(None if t is None else t.data_ptr() for t in pointers), workspace.numel(), n, width, width, 0, width, 2, 2)
        stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
        return lambda: lib.odc_layer_norm_backward(ctypes.byref(call), stream), (mean, rstd, workspace)

    def results(before, after):
        """``before`` and ``after`` every call (torch's own kernels between them would report the error themselves)."""
        ps, ms, vs = [t.clone() for t in starts], [torch.zeros_like(t) for t in starts], [torch.zeros_like(t) for t in starts]
        out = [*ps, *ms, *vs]

        def called(call):
            before()
            result = call()
            after()
            return result

        called(lambda: ops.adamw_step(ps, gs, ms, vs, step=1, lr=1e-2))
        out += [called(lambda: ops.squared_norm(gs)), called(lambda: ops.dequantize_blocks(codes, scales))]
        for x, dy in zip(rows, grads):
            out.append(called(lambda: ops.layer_norm(x, x.shape[1])))
            gradients = [torch.empty_like(x), torch.empty_like(x[0]), torch.empty_like(x[0])]
            call, _kept = backward(x, dy, gradients)
            assert called(call) == 0, lib.odc_ops_last_error()
            out += gradients
        return out

    want = results(lambda: None, lambda: None)
    got = results(lambda: leave_an_error(hip), lambda: hip.hipGetLastError())
    assert len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want))
