"""torch.autocast leaves the norms as they are: the dtype of the input, the same bits."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("autocast", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_autocast_changes_nothing(autocast, dtype):
    from odc_amd import ops

    gen = torch.Generator(device="cuda").manual_seed(0)
    norm = ops.LayerNorm(96).cuda()
    x, r, dy = (torch.randn(50, 96, generator=gen, device="cuda").to(dtype) for _ in range(3))
    results = []
    for enabled in (False, True):
        leaf, other = x.clone().requires_grad_(), r.clone().requires_grad_()
        with torch.autocast("cuda", dtype=autocast, enabled=enabled):
            y, total = norm(leaf, other)
            z = norm(leaf)
        grads = torch.autograd.grad((y, z), (leaf, other, norm.weight, norm.bias), (dy, dy))
        results.append((y, total, z, *grads))
    assert all(a.dtype == b.dtype and torch.equal(a, b) for a, b in zip(*results)) and results[1][0].dtype == dtype


def test_a_branch_in_16_bits_is_cast_to_its_stream():
    from odc_amd import ops

    norm = ops.LayerNorm(96).cuda()
    branch, stream = torch.ones(4, 96, device="cuda").bfloat16(), torch.arange(4.0 * 96, device="cuda").view(4, 96)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        with pytest.raises(TypeError, match="residual: expected the dtype of the input"):
            norm(branch, stream)
        y, total = norm(branch.float(), stream)
    assert y.dtype == total.dtype == torch.float32 and torch.equal(total, stream + 1)
