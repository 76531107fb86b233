"""What the optimizer's state dict holds and reads. No kernel runs: the extension module is stood in for."""

import copy

import pytest
import torch

from odc_amd.ops import optim


class StandIn:
    def __init__(self):
        self.calls = []

    def adamw_prepare(self, *args):
        if any(p.dtype == torch.float64 for p in args[0]):
            raise TypeError("refused")
        return args

    def adamw_launch(self, args):
        self.calls.append(args)


@pytest.fixture
def calls(monkeypatch):
    stand_in = StandIn()
    monkeypatch.setattr(optim, "_host_path", stand_in)
    return stand_in.calls


def parameters(n=3, dtype=torch.float32):
    ps = [torch.nn.Parameter(torch.ones(4 + k, dtype=dtype)) for k in range(n)]
    for p in ps:
        p.grad = torch.ones_like(p)
    return ps


def test_torchs_states_are_read(calls):
    """Three parameters at one step are one call, whose number is an int."""
    ps = parameters()
    theirs = torch.optim.AdamW(ps, lr=0.5, weight_decay=0.25)
    for _ in range(5):
        theirs.step()
    saved = copy.deepcopy(theirs.state_dict())
    assert isinstance(saved["state"][0]["step"], torch.Tensor)
    ours = optim.AdamW(ps)
    ours.load_state_dict(saved)
    ours.step()
    assert len(calls) == 1
    _, _, m, _, v, _, _, _, step, lr, *_ = calls[0]
    assert type(step) is int and step == 6 and lr == 0.5
    for p, a, b in zip(ps, m, v):
        assert torch.equal(a, theirs.state[p]["exp_avg"]) and torch.equal(b, theirs.state[p]["exp_avg_sq"])
        assert type(ours.state[p]["step"]) is int and ours.state[p]["step"] == 6


@pytest.mark.parametrize("bits", [32, 8])
def test_a_refused_step_leaves_no_states(calls, bits):
    ps = parameters(2) + parameters(1, torch.float64)
    opt = optim.AdamW(ps, state_bits=bits)
    with pytest.raises(TypeError):
        opt.step()
    assert not calls and len(opt.state) == 0 and opt.state_dict()["state"] == {}
    ps[2].grad = None
    opt.step()
    assert len(opt.state) == 2
    again = optim.AdamW(ps, state_bits=bits)
    again.load_state_dict(copy.deepcopy(opt.state_dict()))
    assert again.state[ps[0]]["step"] == again.state[ps[1]]["step"] == 1


@pytest.mark.parametrize("bits", [32, 8])
def test_a_state_that_was_only_looked_at(calls, bits):
    """``opt.state`` makes an empty state for who asks; it is saved, and no state to the optimizer that reads it."""
    ps = parameters()
    opt = optim.AdamW(ps, state_bits=bits)
    opt.step()
    ps.append(torch.nn.Parameter(torch.ones(9)))
    opt.add_param_group({"params": ps[3:]})
    assert opt.state[ps[3]] == {}
    saved = copy.deepcopy(opt.state_dict())
    assert {} in saved["state"].values()
    again = optim.AdamW([{"params": ps[:3]}, {"params": ps[3:]}], state_bits=bits)
    again.load_state_dict(saved)
    ps[3].grad = torch.ones(9)
    again.step()
    assert [again.state[p]["step"] for p in ps] == [2, 2, 2, 1]


@pytest.mark.parametrize("kind,option", [("AdamW", dict(maximize=True)), ("AdamW", dict(amsgrad=True)), ("Adam", dict(weight_decay=0.1)),
                                         ("Adam", dict(maximize=True))])
def test_options_that_change_the_step_are_refused(calls, kind, option):
    """They came with the parameter groups, and were ignored."""
    ps = parameters()
    theirs = getattr(torch.optim, kind)(ps, **option)
    theirs.step()
    with pytest.raises(ValueError, match="another optimizer"):
        optim.AdamW(ps).load_state_dict(theirs.state_dict())


def test_adam_without_decay_is_read(calls):
    ps = parameters()
    theirs = torch.optim.Adam(ps)
    theirs.step()
    ours = optim.AdamW(ps)
    ours.load_state_dict(theirs.state_dict())
    ours.step()
    assert calls[0][13] == 0 and calls[0][8] == 2  # no decay, the second step
