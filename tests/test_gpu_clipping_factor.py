"""The factor that clips the gradients is rounded once in its root and once in its division: the nearest fp32 numbers.
(It multiplies every gradient of a step: a unit of its last place is an error that all of them share.)"""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("scale", [1.0, 0.25])
def test_the_factor_is_the_nearest_number(eight, scale):
    """With beta1 = 0 and a gradient of one m is the factor itself: read from the parameter's step where states have 8 bits."""
    from odc_amd import ops

    gen = torch.Generator(device="cuda").manual_seed(0)
    norms = torch.exp2(torch.rand(200, generator=gen, device="cuda") * 60 - 10)
    got = []
    for norm in norms:
        p, g, m, v = (torch.full((1,), float(k), device="cuda") for k in (0, 1, 0, 0))
        numbers = dict(step=1, betas=(0.0, 0.0), grad_scale=scale, squared_norm=norm, max_norm=1.0)
        if eight:
            codes = [torch.zeros(1, dtype=torch.uint8, device="cuda").view(d) for d in (torch.float8_e4m3fn, torch.float8_e8m0fnu) * 2]
            # p = -lr m / (|g| + 2^60), whose sum and reciprocal are 2^60 and 2^-60
            ops.adamw_step_8bit([p], [g], *([c] for c in codes), lr=2.0**60, eps=2.0**60, seed=0, **numbers)
            got.append(-p)
        else:
            ops.adamw_step([p], [g], [m], [v], lr=0.0, **numbers)
            got.append(m)
    norm = norms.cpu().numpy()
    root = np.sqrt(norm) * np.float32(scale)  # (a power of two: exact)
    assert root.dtype == np.float32
    want = np.minimum(np.float32(1), np.float32(1) / (root + np.float32(1e-6))) * np.float32(scale)
    assert want.dtype == np.float32
    assert np.array_equal(torch.cat(got).cpu().numpy(), want)
