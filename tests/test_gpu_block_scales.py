"""States in 8 bits with every scale that E8M0 has: 0 is 2^-127 and 255 is not a number, as torch reads them."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def every_code_and_scale(device="cuda"):
    """Blocks of the 256 codes, eight to a scale."""
    scales = torch.arange(256, dtype=torch.uint8, device=device).repeat_interleave(8)
    codes = torch.arange(256, dtype=torch.uint8, device=device).repeat(256)
    return codes.view(torch.float8_e4m3fn), scales.view(torch.float8_e8m0fnu)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cut", [0, 13])
def test_all_codes_with_all_scales(dtype, cut):
    from odc_amd import ops

    codes, scales = every_code_and_scale()
    codes = codes[: codes.numel() - cut]  # a vector that is not whole, at the end
    got = ops.dequantize_blocks(codes, scales, dtype)
    # (from the bytes, so that nothing but powers of two is asked of torch)
    powers = torch.exp2(scales.view(torch.uint8).double() - 127)
    powers[scales.view(torch.uint8) == 255] = float("nan")
    want = (codes.double() * powers.repeat_interleave(32)[: codes.numel()]).float().to(dtype)
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got[~want.isnan()], want[~want.isnan()])
    exact = codes.double() * powers.repeat_interleave(32)[: codes.numel()]
    number = scales.view(torch.uint8).repeat_interleave(32)[: codes.numel()]
    inside = ~want.isnan() & (number <= 246) & (number >= (3 if dtype == torch.bfloat16 else 0))
    if dtype != torch.float16:
        assert torch.equal(got[inside].double(), exact[inside])


@pytest.mark.parametrize("scale", [0, 1, 254, 255])
def test_a_step_reads_them_so(scale):
    """An average of zero gradient is beta1 times what it was: m itself is read back from the parameter's step."""
    from odc_amd import ops

    n = 64
    codes = torch.full((n,), 0x38, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)  # 1.0
    scales = torch.full((2,), scale, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu)
    roots, root_scales = (torch.zeros(k, dtype=torch.uint8, device="cuda") for k in (n, 2))
    p = torch.zeros(n, device="cuda")
    ops.adamw_step_8bit([p], [torch.zeros(n, device="cuda")], [codes], [scales], [roots.view(torch.float8_e4m3fn)],
                        [root_scales.view(torch.float8_e8m0fnu)], step=1, lr=0.5, betas=(0.5, 0.5), eps=1.0, seed=0)
    # p = -lr / (1 - beta1) * beta1 m / eps = -m / 2
    want = -0.5 * 2.0 ** (scale - 127) if scale < 255 else float("nan")
    if scale == 255:
        assert bool(p.isnan().all())
    else:
        assert bool((p == want).all()), (float(p[0]), want)


def test_states_to_begin_with_stay_zeros():
    """All zeros, scales included: zero codes are zeros whatever 2^-127 is."""
    from odc_amd import ops

    codes, scales = (torch.zeros(k, dtype=torch.uint8, device="cuda") for k in (100, 4))
    assert not bool(ops.dequantize_blocks(codes.view(torch.float8_e4m3fn), scales.view(torch.float8_e8m0fnu)).any())
