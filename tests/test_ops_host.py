"""The host side of libodc_ops.so without a GPU: the C ABI's surface, its checks and launch plans under
AddressSanitizer and UBSan, the refusal of what is not on a GPU, and the optimizer's arguments."""

import re
import subprocess
from pathlib import Path

import pytest
import torch

from odc_amd import _native, ops

ROOT = Path(__file__).resolve().parent.parent
CSRC = ROOT / "odc_amd" / "csrc"


def test_every_declared_symbol_is_there():
    header = (ROOT / "include" / "odc_ops.h").read_text()
    declared = set(re.findall(r"^\w[\w\s\*]*?\b(odc_[a-z_0-9]+)\(", header, re.M))
    assert declared == set(_native.OPS_EXPORTED_SYMBOLS)
    _native.load_ops()
    assert all(hasattr(_native._ops_lib, name) for name in declared)
    version = int(re.search(r"ODC_OPS_ABI_VERSION (\d+)", header).group(1))
    assert _native._ops_lib.odc_ops_abi_version() == _native.OPS_ABI_VERSION == version


def test_the_header_is_plain_c():
    subprocess.run(["gcc", "-std=c99", "-fsyntax-only", "-Wall", "-Wextra", "-pedantic", "-x", "c", str(ROOT / "include" / "odc_ops.h")],
                   check=True)


def test_checks_and_plans_under_asan_and_ubsan(tmp_path):
    exe = tmp_path / "check"
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-fno-sanitize-recover=all", "-Wall", "-Wextra", "-Werror",
                    "-Wno-missing-field-initializers", "-Wno-unknown-pragmas", f"-I{ROOT / 'include'}", f"-I{CSRC}", str(CSRC / "odc_ops_host.cpp"),
                    str(ROOT / "tests" / "cpu" / "no_ops_device.cpp"), "-o", str(exe)], check=True)
    proc = subprocess.run([str(exe)], capture_output=True, text=True)
    assert proc.returncode == 0 and proc.stdout == "ok\n", proc.stdout + proc.stderr


def test_the_host_side_needs_no_hip_header():
    text = (CSRC / "odc_ops_host.cpp").read_text()
    assert "hip/hip_runtime" not in text and "__global__" not in text and "hipLaunch" not in text


def test_a_stale_extension_is_refused():
    with pytest.raises(ImportError, match="is stale"):
        _native._load_torch_binding_file(_native.OPS_BINDING_PATH, "odc_ops_torch", 99)


def test_tensors_of_the_cpu_are_refused():
    x = torch.randn(4, 8)
    with pytest.raises(TypeError, match="GPU"):
        ops.layer_norm(x, 8)
    with pytest.raises(TypeError, match="GPU"):
        ops.add_layer_norm(x, x, 8)
    with pytest.raises(TypeError, match="GPU"):
        ops.LayerNorm(8)(x)
    with pytest.raises(TypeError, match="GPU"):
        ops.squared_norm([x])
    with pytest.raises(TypeError, match="GPU"):
        ops.adamw_step([x], [x], [x], [x], step=1, lr=1e-3)
    with pytest.raises(TypeError, match="GPU"):
        ops.dequantize_blocks(x.to(torch.float8_e4m3fn), x.to(torch.float8_e8m0fnu))


def test_what_is_no_list_is_refused():
    x = torch.randn(4)
    with pytest.raises(TypeError, match="sequence"):
        ops.adamw_step(5, [x], [x], [x], step=1, lr=1e-3)
    with pytest.raises(TypeError):
        ops.squared_norm(5)
    with pytest.raises(TypeError, match="torch.Tensor"):
        ops.squared_norm([5])
    with pytest.raises(ValueError, match="no tensors"):
        ops.squared_norm(iter([]))


def test_optimizer_arguments():
    p = torch.nn.Parameter(torch.ones(3))
    opt = ops.AdamW([p], lr=0.5, betas=(0.8, 0.9), eps=1e-6, weight_decay=0.0, state_bits=8, max_norm=1.0, seed=3)
    assert opt.param_groups[0]["lr"] == 0.5 and opt.param_groups[0]["betas"] == (0.8, 0.9)
    for wrong in (dict(lr=-1.0), dict(eps=-1.0), dict(weight_decay=-1.0), dict(betas=(1.0, 0.9)), dict(state_bits=16), dict(max_norm=-1.0)):
        with pytest.raises(ValueError):
            ops.AdamW([p], **wrong)
    opt.step()  # nothing has a gradient
    assert not opt.state[p]
    with pytest.raises(ValueError, match="nothing to clip"):
        ops.AdamW([p]).step(squared_norm=torch.ones(()))


def test_the_package_does_not_need_the_operators():
    """``import odc_amd`` loads the primitives alone; the operators come with ``odc_amd.ops``."""
    code = "import odc_amd, sys; assert 'odc_amd.ops' not in sys.modules; from odc_amd import ops; assert ops.AdamW"
    import sys

    subprocess.run([sys.executable, "-c", code], check=True, cwd=ROOT)
