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
