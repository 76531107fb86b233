"""A step of odc_amd.ops.AdamW makes a call for each group and dtype. One that is refused has made none of them."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from odc_amd import ops

    assert torch.cuda.is_available(), "GPU test run without a GPU"
    return ops


def parameters(*dtypes):
    gen = torch.Generator(device="cuda").manual_seed(0)
    ps = [torch.nn.Parameter(torch.randn(300 + k, generator=gen, device="cuda").to(d)) for k, d in enumerate(dtypes)]
    for p in ps:
        p.grad = torch.randn(p.shape, generator=gen, device="cuda").to(p.dtype)
    return ps


def everything(ps, opt):
    """Bits of parameters and states, version counters, step numbers."""
    bits = [t.detach().clone().view(torch.uint8) for p in ps for t in (p, *(v for v in opt.state.get(p, {}).values() if isinstance(v, torch.Tensor)))]
    return bits, [p._version for p in ps], [opt.state.get(p, {}).get("step") for p in ps]


def same(a, b):
    return len(a[0]) == len(b[0]) and all(torch.equal(x, y) for x, y in zip(a[0], b[0])) and a[1:] == b[1:]


def refused_by_dtype(opt, ps):
    ps[1].data = ps[1].data.half()
    ps[1].grad = ps[1].data.clone()
    return TypeError


def refused_by_number(opt, ps):
    opt.param_groups[1]["lr"] = -1.0
    return RuntimeError


def refused_by_state(opt, ps):
    if ps[1] in opt.state:
        name = "exp_avg"
        opt.state[ps[1]][name] = opt.state[ps[1]][name][:5]
    else:
        opt.param_groups[1]["betas"] = (0.9, 2.0)
    return (ValueError, RuntimeError)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("steps", [0, 2])
@pytest.mark.parametrize("spoil", [refused_by_dtype, refused_by_number, refused_by_state])
def test_a_refused_step_has_written_nothing(ops, bits, steps, spoil):
    ps = parameters(torch.float32, torch.float32, torch.bfloat16)
    opt = ops.AdamW([{"params": [p]} for p in ps], lr=0.1, state_bits=bits)
    for _ in range(steps):
        opt.step()
    error = spoil(opt, ps)
    before = everything(ps, opt)
    with pytest.raises(error):
        opt.step()
    assert same(before, everything(ps, opt))


@pytest.mark.parametrize("bits", [32, 8])
def test_a_step_behind_a_refused_one(ops, bits):
    """The step that follows is the one that would have been made."""
    results = []
    for refused in (False, True):
        ps = parameters(torch.float32, torch.bfloat16)
        opt = ops.AdamW([{"params": [ps[0]]}, {"params": [ps[1]], "lr": 0.2}], lr=0.1, state_bits=bits)
        for _ in range(3):
            if refused:
                opt.param_groups[1]["lr"] = float("nan")
                with pytest.raises(RuntimeError):
                    opt.step()
                opt.param_groups[1]["lr"] = 0.2
            opt.step()
        results.append(everything(ps, opt))
    assert same(*results)


def test_a_prepared_call_is_the_call(ops):
    """The steps of the class are those of the function."""
    ps = parameters(torch.float32)
    twin, m, v = ps[0].detach().clone(), torch.zeros_like(ps[0].data), torch.zeros_like(ps[0].data)
    opt = ops.AdamW(ps, lr=0.1, weight_decay=0.1)
    for step in (1, 2):
        opt.step()
        ops.adamw_step([twin], [ps[0].grad], [m], [v], step=step, lr=0.1, weight_decay=0.1)
    assert torch.equal(twin, ps[0]) and torch.equal(m, opt.state[ps[0]]["exp_avg"]) and torch.equal(v, opt.state[ps[0]]["exp_avg_sq"])
