"""odc_amd.ops.squared_norm has no derivative, and says so to a backward pass that comes by."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtypes", [(torch.float32, torch.float32), (torch.float32, torch.bfloat16)])
def test_a_derivative_is_refused_and_not_zero(dtypes):
    from odc_amd import ops

    w = [torch.ones(100, dtype=d, device="cuda", requires_grad=True) for d in dtypes]
    x = torch.zeros(50, device="cuda", requires_grad=True)
    penalty = ops.squared_norm(w)
    assert float(penalty.detach()) == 200 and penalty.requires_grad and penalty.shape == ()
    with pytest.raises(RuntimeError, match="squared_norm"):
        (x.sum() + penalty).backward()
    with pytest.raises(RuntimeError, match="squared_norm"):
        torch.autograd.grad(ops.squared_norm([t * 2 for t in w]), w[0])
    assert w[0].grad is None


def test_what_asks_for_none_has_none():
    from odc_amd import ops

    w = torch.ones(100, device="cuda", requires_grad=True)
    with torch.no_grad():
        assert not ops.squared_norm([w]).requires_grad
    (w * 3).sum().backward()
    total = ops.squared_norm([w.grad, w.detach()])
    assert not total.requires_grad and float(total) == 1000
    optimizer = ops.AdamW([w], max_norm=1.0)
    optimizer.step(squared_norm=ops.squared_norm([w]))  # a number with a graph behind it is a number
    assert float(w.detach()[0]) < 1
