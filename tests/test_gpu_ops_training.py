"""The operators of odc_amd.ops together, as a training program runs them: in the transformer example under torch's
``fully_shard``, and on the shards of an arena that gathers read afterwards."""

import re
import subprocess
import sys
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu
SCRIPT = Path(__file__).resolve().parent.parent / "examples" / "fsdp2_toy.py"


def run(*args):
    proc = subprocess.run([sys.executable, str(SCRIPT), "--steps", "6", *args], capture_output=True, text=True, timeout=300)
    assert proc.returncode == 0, proc.stdout[-2000:] + proc.stderr[-2000:]
    losses = [float(x) for x in re.findall(r"loss ([0-9.]+)  gradient shards match", proc.stdout)]
    assert len(losses) == 6, proc.stdout
    return losses


@pytest.mark.parametrize("extra", [(), ("--state-bits", "8"), ("--mixed-precision",), ("--mixed-precision", "--state-bits", "8", "--world-size", "3")])
def test_the_example_trains_with_the_operators(extra):
    """Every step's gradient shards match the unsharded twin's bit for bit (the script fails otherwise)."""
    losses = run("--native-ops", *extra)
    assert losses[-1] < losses[0]


def test_the_first_loss_is_that_of_the_example_without_them():
    """The same model, weights and batch: the norms differ by roundings of fp32, in a loss of about 7 printed to 1e-4."""
    assert abs(run("--native-ops")[0] - run()[0]) < 5e-4


def test_a_gather_behind_the_step_reads_the_new_parameters(make_world):
    """Shards in the symmetric arena, stepped in place with their bf16 copies: a gather of either sees the step. Nothing
    but stream order lies between them."""
    import odc_amd as odc
    from odc_amd import ops

    W, n = 4, 30_011
    group = make_world(W, 8 << 20)
    registry = odc.SymmBufferRegistry.get_instance()
    gen = torch.Generator(device="cuda").manual_seed(0)
    registry.allocate_symm_buffer("p", (n,), torch.float32)
    registry.allocate_symm_buffer("p16", (n,), torch.bfloat16)
    shards, copies = registry.peer_tensors["p"], registry.peer_tensors["p16"]
    for s in shards:
        s.copy_(torch.randn(n, generator=gen, device="cuda"))
    grads = [torch.randn(n, generator=gen, device="cuda") for _ in range(W)]
    ms, vs = ([torch.zeros(n, device="cuda") for _ in range(W)] for _ in range(2))
    want = [s.clone() for s in shards]
    reference = torch.optim.AdamW([torch.nn.Parameter(w) for w in want], lr=1e-2, weight_decay=0.1, eps=1e-8)
    out, out16 = torch.empty(W * n, device="cuda"), torch.empty(W * n, dtype=torch.bfloat16, device="cuda")
    gather = odc.GatherService()
    for step in (1, 2):
        ops.adamw_step(shards, grads, ms, vs, step=step, lr=1e-2, weight_decay=0.1, copies=copies)
        gather.gather_into_tensor(out, registry.get_symm_buffer("p"), group)
        gather.gather_into_tensor(out16, registry.get_symm_buffer("p16"), group)
        for p, g in zip(reference.param_groups[0]["params"], grads):
            p.grad = g
        reference.step()
        full = torch.cat([p.detach() for p in reference.param_groups[0]["params"]])
        assert float((out - full).abs().max()) < 1e-5
        assert torch.equal(out16, out.bfloat16())


def test_sharded_parameters_need_the_norm_of_all_ranks():
    """DTensor parameters of a mesh of more than one rank: their own norm is not the model's, and clipping by it is
    refused (in a child process: the process group is the child's own)."""
    code = """
import torch, torch.distributed as dist
from torch.distributed.device_mesh import init_device_mesh
from torch.distributed.tensor import DTensor, Shard
from torch.testing._internal.distributed.fake_pg import FakeStore
from odc_amd import ops
dist.init_process_group("fake", rank=0, world_size=2, store=FakeStore())
mesh = init_device_mesh("cuda", (2,))
p = torch.nn.Parameter(DTensor.from_local(torch.ones(8, 4, device="cuda"), mesh, [Shard(0)], run_check=False))
p.grad = DTensor.from_local(torch.full((8, 4), 2.0, device="cuda"), mesh, [Shard(0)], run_check=False)
for bits in (32, 8):
    opt = ops.AdamW([p], lr=0.1, max_norm=1.0, state_bits=bits)
    try:
        opt.step()
    except ValueError as e:
        assert "shards" in str(e)
    else:
        raise SystemExit("clipped by a shard's norm")
    before, version = p._local_tensor.clone(), p._version
    opt.step(squared_norm=2 * ops.squared_norm([p.grad._local_tensor]))
    assert not torch.equal(before, p._local_tensor) and p._version > version
    assert opt.state[p]["step"] == 1
print("ok")
"""
    proc = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300, cwd=SCRIPT.parent.parent)
    assert proc.returncode == 0 and "ok" in proc.stdout, proc.stdout + proc.stderr[-2000:]
