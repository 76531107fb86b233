"""The mean of a row is right to a rounding or two whatever the row's length: rows of one value come out as zeros, and the
bounds do not grow with the length.

Bounds. u = 2^-24, M = max|x|, a = M / sigma. The mean is off by at most 4 u M (in rows in registers by u M and 64 u of what
the values differ by), so x - mean is off by 4 u M and a rounding, the variance by twice that relative to sigma and by less
than 64 roundings of its own: a value of z by less than (16 u a + 128 u (1 + |z|)) (1 + |z|)."""

import pytest
import torch

U = 2.0**-24
pytestmark = pytest.mark.gpu
# less than a vector, registers of 16 to 1024 lanes, one to four vectors each, the passes over wide rows
WIDTHS = [1, 2, 3, 5, 7, 33, 96, 257, 1001, 2500, 4099, 8200, 14336, 16384, 16389, 20001, 33000, 100_003]


@pytest.fixture(scope="module")
def ops():
    from odc_amd import ops

    assert torch.cuda.is_available(), "GPU test run without a GPU"
    return ops


@pytest.mark.parametrize("width", WIDTHS + [1 << 20, (1 << 26) - 3])
@pytest.mark.parametrize("dtype,values", [(torch.float32, (0.1, 1.1, -3.3, 1e9, 1e-12)), (torch.float16, (0.1, 60000.0)), (torch.bfloat16, (0.1, -1.1))])
def test_rows_of_one_value_are_zeros(ops, width, dtype, values):
    """No element differs from the mean, and eps alone is divided by."""
    for value in values if width < 1 << 26 else values[:2]:
        x = torch.full((3 if width < 1 << 20 else 1, width), value, device="cuda").to(dtype)
        assert not bool(ops.layer_norm(x, width).any()), value
        if width < 1 << 20 and dtype != torch.float16:
            y, total = ops.add_layer_norm(x, x, width)
            assert torch.equal(total, x + x) and not bool(y.any()), value


@pytest.mark.parametrize("width", WIDTHS + [1 << 22])
@pytest.mark.parametrize("offset", [0.0, 100.0, 30000.0])
@pytest.mark.parametrize("pad", [0, 1])
def test_bounds_that_do_not_grow_with_the_row(ops, width, offset, pad):
    gen = torch.Generator(device="cuda").manual_seed(width)
    rows = 5 if width < 1 << 20 else 1
    x = (torch.randn(rows, width + pad, generator=gen, device="cuda") * 1.5 + offset)[:, :width].requires_grad_()
    w = (1 + 0.2 * torch.randn(width, generator=gen, device="cuda")).requires_grad_()
    dy = torch.randn(rows, width, generator=gen, device="cuda")
    y = ops.layer_norm(x, width, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    v, h = x.detach().double(), dy.double() * w.detach().double()
    mean = v.mean(1, keepdim=True)
    sigma = ((v - mean).square().mean(1, keepdim=True) + 1e-5).sqrt()
    z = (v - mean) / sigma
    ez = (16 * U * v.abs().amax(1, keepdim=True) / sigma + 128 * U * (1 + z.abs())) * (1 + z.abs())
    off = (y.detach().double() - z * w.detach().double()).abs()
    assert bool((off <= (ez + 4 * U * z.abs()) * w.detach().double().abs()).all()), float((off / ez).max())
    mh, mz = h.abs().mean(1, keepdim=True), (h * z).abs().mean(1, keepdim=True)
    want = (h - h.mean(1, keepdim=True) - z * (h * z).mean(1, keepdim=True)) / sigma
    edx = (8 * U * (h.abs() + z.abs() * mz) + 64 * U * (mh + z.abs() * mz) + ez * mz + z.abs() * (h.abs() * ez).mean(1, keepdim=True)) / sigma * 2
    # the reciprocal of sigma carries the variance's error into all of it
    edx = edx + want.abs() * ez.amin(1, keepdim=True)
    off = (dx.double() - want).abs()
    assert bool((off <= edx + 2.0**-149).all()), float((off / edx).max())
    off = (dw.double() - (dy.double() * z).sum(0)).abs()
    assert bool((off <= (dy.double().abs() * (ez + 8 * U * z.abs())).sum(0) + 2.0**-149).all())
