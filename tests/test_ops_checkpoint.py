"""The optimizer's states through torch's distributed checkpoint, and shards that need the norm of all ranks, on two
ranks of the CPU. The kernels are stood in for
by a step that writes rank and place into every state."""

import itertools

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

MARK = {"exp_avg": 16, "exp_avg_scale": 32, "exp_avg_sq": 48, "exp_avg_root": 48, "exp_avg_root_scale": 64}


class StandIn:
    """For the extension module: ``adamw_launch`` writes into the state of tensor k on rank r, list l: 16 l + 8 r + k."""

    def adamw_prepare(self, params, grads, *rest):
        lists = rest[:4]
        for one, per in zip(lists, (1, 32, 1, 32)):
            for t, p in zip(one or (), params):
                assert t.is_contiguous() and t.numel() == -(-p.numel() // per)
        return lists

    def adamw_launch(self, lists):
        for number, one in enumerate(lists):
            for k, t in enumerate(one or ()):
                value = 16 * (number + 1) + 8 * dist.get_rank() + k
                t.view(torch.uint8).fill_(value) if t.element_size() == 1 else t.fill_(value)

    def squared_norm(self, tensors):
        return torch.stack([t.square().sum() for t in tensors]).sum()


def local(t):
    return getattr(t, "_local_tensor", t)


def numbers(t):
    return local(t).view(torch.uint8) if t.element_size() == 1 else local(t)


class Model(torch.nn.Module):
    def __init__(self, mesh, shapes, dim):
        from torch.distributed.tensor import Shard, distribute_tensor

        super().__init__()
        self.p = torch.nn.ParameterList(
            torch.nn.Parameter(distribute_tensor(torch.ones(shape), mesh, [Shard(min(dim, len(shape) - 1))])) for shape in shapes)


def stepped(mesh, shapes, dim=0, **arguments):
    from odc_amd.ops import optim

    model = Model(mesh, shapes, dim)
    opt = optim.AdamW(model.parameters(), **arguments)
    for p in model.parameters():
        p.grad = torch.ones_like(p)
    opt.step()
    return model, opt


def fresh(mesh, shapes, dim=0, **arguments):
    from odc_amd.ops import optim

    model = Model(mesh, shapes, dim)
    return model, optim.AdamW(model.parameters(), **arguments)


def save(model, opt, path):
    import torch.distributed.checkpoint as dcp
    from torch.distributed.checkpoint.state_dict import get_optimizer_state_dict

    dcp.save(get_optimizer_state_dict(model, opt), checkpoint_id=path)


def load(model, opt, path):
    import torch.distributed.checkpoint as dcp
    from torch.distributed.checkpoint.state_dict import get_optimizer_state_dict, set_optimizer_state_dict

    state = get_optimizer_state_dict(model, opt)
    dcp.load(state, checkpoint_id=path)
    set_optimizer_state_dict(model, opt, state)


def restored(rank, mesh, path, bits, shapes, dim=0, **arguments):
    """What rank ``rank`` wrote is what it reads."""
    save(*stepped(mesh, shapes, dim, state_bits=bits), path)
    model, opt = fresh(mesh, shapes, dim, state_bits=bits, **arguments)
    load(model, opt, path)
    for k, p in enumerate(model.parameters()):
        state = opt.state[p]
        assert state["step"] == 1 and type(state["step"]) is int
        for name, value in state.items():
            if name != "step" and local(p).numel():
                n = -(-local(p).numel() // (32 if "scale" in name else 1))
                assert bool((numbers(value).reshape(-1)[:n] == MARK[name] + 8 * rank + k).all()), (rank, k, name)
    for p in model.parameters():
        p.grad = torch.zeros_like(p)
    opt.step()  # the lists of a step have the lengths of the shards (StandIn)
    assert all(opt.state[p]["step"] == 2 for p in model.parameters())


def another_sharding(rank, mesh, path):
    """States in 8 bits belong to their shard's blocks: read for another sharding they are refused."""
    save(*stepped(mesh, [(8, 64)], 0, state_bits=8), path)
    model, opt = fresh(mesh, [(8, 64)], 1, state_bits=8)
    with pytest.raises(BaseException, match="Size mismatch"):
        load(model, opt, path)


def child(rank, directory, body, arguments):
    from torch.distributed.device_mesh import init_device_mesh

    from odc_amd.ops import optim

    optim._host_path = StandIn()
    dist.init_process_group("gloo", rank=rank, world_size=2, init_method=f"file://{directory}/rendezvous")
    try:
        body(rank, init_device_mesh("cpu", (2,)), f"{directory}/checkpoint", *arguments)
    finally:
        dist.destroy_process_group()


def on_two_ranks(tmp_path, body, *arguments):
    mp.spawn(child, (str(tmp_path), body, arguments), nprocs=2)


# even shards, shards of different lengths, blocks that end inside a row, shards along the second dimension
@pytest.mark.parametrize("bits,dim", itertools.product((32, 8), (0, 1)))
def test_every_rank_reads_what_it_wrote(tmp_path, bits, dim):
    on_two_ranks(tmp_path, restored, bits, [(8, 32), (7, 33), (101,), (64,)], dim)


def test_states_in_8_bits_are_not_read_for_another_sharding(tmp_path):
    on_two_ranks(tmp_path, another_sharding)


def own_norm(rank, mesh, path):
    """A step of torch's own that begins the states has zero gradients, and needs no norm; with others it does, on a rank
    whose gradients are not zero."""
    restored(rank, mesh, path, 32, [(8, 32), (101,)], max_norm=1.0)
    restored(rank, mesh, path + "8", 8, [(8, 32), (101,)], max_norm=1.0)
    model, opt = fresh(mesh, [(8, 32), (101,)], max_norm=1.0)
    p, q = model.parameters()
    p.grad, q.grad = torch.zeros_like(p), torch.zeros_like(q)
    q.grad._local_tensor[-1] = 1e-30  # its square is no fp32 number
    with pytest.raises(ValueError, match="shards"):
        opt.step()
    q.grad._local_tensor[-1] = float("nan")
    with pytest.raises(ValueError, match="shards"):
        opt.step()


def test_clipped_shards_are_resumed(tmp_path):
    on_two_ranks(tmp_path, own_norm)


@pytest.mark.parametrize("bits", [32, 8])
def test_a_rank_whose_shard_is_empty(tmp_path, bits):
    """One row over two ranks: the second has nothing of it, and states like the first."""
    on_two_ranks(tmp_path, restored, bits, [(8, 32), (1, 32)])


def flat_parameters(rank, mesh, path):
    from torch.distributed.fsdp import FullyShardedDataParallel as FSDP

    from odc_amd.ops import optim

    model = FSDP(torch.nn.Linear(7, 5), device_id=torch.device("cpu"), use_orig_params=False)
    flat, = model.parameters()
    assert flat.numel() == 20
    opt = optim.AdamW([flat], max_norm=1.0)
    flat.grad = torch.ones_like(flat)
    with pytest.raises(ValueError, match="shards"):
        opt.step()
    opt.step(squared_norm=torch.tensor(40.0))
    optim.AdamW([flat]).step()  # without clipping there is nothing to know


def test_flat_shards_need_the_norm_of_all_ranks(tmp_path):
    """FSDP1: clipped by its own norm, every rank would take another step."""
    on_two_ranks(tmp_path, flat_parameters)
