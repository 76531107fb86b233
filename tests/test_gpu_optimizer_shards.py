"""odc_amd.ops.AdamW on DTensor parameters (in child processes: the process group is the child's own)."""

import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parent.parent

PRELUDE = """
import torch, torch.distributed as dist
from torch.distributed.device_mesh import init_device_mesh
from torch.distributed.tensor import DTensor, Shard
from torch.testing._internal.distributed.fake_pg import FakeStore
from odc_amd import ops
rank = {rank}
dist.init_process_group("fake", rank=rank, world_size=2, store=FakeStore())
mesh = init_device_mesh("cuda", (2,))
gen = torch.Generator(device="cuda").manual_seed(rank)
def sharded(shape, dim=0):
    parts = torch.empty(shape, device="meta").chunk(2, dim)
    local = torch.randn(parts[rank].shape if rank < len(parts) else [0 if d == dim else n for d, n in enumerate(shape)], generator=gen, device="cuda")
    stride = torch.empty(shape, device="meta").stride()
    return DTensor.from_local(local, mesh, [Shard(dim)], run_check=False, shape=torch.Size(shape), stride=stride)
"""


def run(rank, code):
    proc = subprocess.run([sys.executable, "-c", PRELUDE.format(rank=rank) + code], capture_output=True, text=True, timeout=100, cwd=ROOT)
    assert proc.returncode == 0 and proc.stdout.endswith("ok\n"), proc.stdout + proc.stderr[-2000:]


@pytest.mark.parametrize("rank", [0, 1])
def test_a_shard_is_stepped_as_a_tensor_of_its_own(rank):
    """Parameters and states have the bits that an optimizer of the local tensors gives them: shards of one length and of
    different ones, along both dimensions."""
    run(rank, """
ps = [torch.nn.Parameter(sharded(shape, dim)) for shape, dim in (((8, 32), 0), ((7, 33), 0), ((101,), 0), ((5, 70), 1))]
twins = [torch.nn.Parameter(p._local_tensor.clone()) for p in ps]
for bits in (8, 32):
    opt, other = (ops.AdamW(x, lr=0.1, state_bits=bits, seed=3) for x in (ps, twins))
    for step in range(3):
        for p, q in zip(ps, twins):
            q.grad = torch.randn(q.shape, generator=gen, device="cuda")
            p.grad = DTensor.from_local(q.grad.clone(), mesh, p.placements, run_check=False, shape=p.shape, stride=p.stride())
        opt.step()
        other.step()
        for p, q in zip(ps, twins):
            assert torch.equal(p._local_tensor, q)
            for name, value in other.state[q].items():
                if name == "step":
                    continue
                mine = opt.state[p][name]
                assert isinstance(mine, DTensor)
                assert torch.equal(mine._local_tensor.reshape(-1)[: value.numel()].view(torch.uint8), value.reshape(-1).view(torch.uint8)), name
            if bits == 8:
                read = [ops.dequantize_blocks(o.state[x]["exp_avg"], o.state[x]["exp_avg_scale"]).reshape(-1)[: q.numel()]
                        for o, x in ((opt, p), (other, q))]
                assert torch.equal(*read) and bool(read[0].any())
print("ok")
""")
