"""The operators where sizes matter: what is streamed past the caches (a pass over more than 256 MB), and offsets that
pass 32 bits, in elements and in bytes. Compared with 64 bits at the ends, in the middle and at the places that 32 bits
would confuse; the bounds are those of tests/test_gpu_layer_norm.py and tests/test_gpu_adamw.py."""

import pytest
import torch

from tests.test_gpu_adamw import NUMBERS, formula, mixed, neighbours
from tests.test_gpu_layer_norm import U, close, reference, z_error

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from odc_amd import ops

    assert torch.cuda.is_available(), "GPU test run without a GPU"
    yield ops
    torch.cuda.empty_cache()


def randn(shape, dtype, gen, scale=1.0, offset=0.0):
    """Filled in parts: a part's fp32 is all there is beside the result."""
    out = torch.empty(shape, dtype=dtype, device="cuda")
    flat = out.view(-1)
    for a in range(0, flat.numel(), 1 << 28):
        n = min(1 << 28, flat.numel() - a)
        flat[a : a + n].copy_(torch.randn(n, generator=gen, device="cuda").mul_(scale).add_(offset))
    return out


@pytest.mark.parametrize("rows,width,dtype,add", [
    (30_000, 4096, torch.bfloat16, False),   # a row to half of a workgroup, streamed
    (9_000, 14_336, torch.bfloat16, True),   # two vectors to a lane, weights in LDS, streamed
    (6_000, 16_384, torch.float32, False),   # four
    (20_000, 4095, torch.float16, True),     # ragged: at any alignment
    (5_000, 40_000, torch.bfloat16, False),  # wider than the registers
    (600_000, 4096, torch.bfloat16, False),  # 2.5 G elements
])
def test_layer_norm(ops, rows, width, dtype, add):
    gen = torch.Generator(device="cuda").manual_seed(rows)
    x = randn((rows, width), dtype, gen, 1.5, 0.3).requires_grad_()
    r = randn((rows, width), dtype, gen).requires_grad_() if add else None
    w = (1 + 0.2 * torch.randn(width, generator=gen, device="cuda")).requires_grad_()
    b = (0.2 * torch.randn(width, generator=gen, device="cuda")).requires_grad_()
    dy = randn((rows, width), dtype, gen, 0.1)
    if add:
        y, total = ops.add_layer_norm(x, r, width, w, b)
        dx, dw, db = torch.autograd.grad((y, total), (x, w, b), (dy, dy))
        normalised = total.detach()
    else:
        y = ops.layer_norm(x, width, w, b)
        dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
        normalised = x.detach()
    confused = (1 << 32) // (width * x.element_size()), (1 << 31) // width, (1 << 32) // width
    some = sorted({i + d for i in (0, rows // 2, rows - 1, *confused) for d in (-2, -1, 0, 1, 2) if 0 <= i + d < rows})
    n, d = normalised[some], dy[some]
    want_y, z, sigma, want_dx, _, _, h = reference(n, w.detach(), b.detach(), 1e-5, d)
    ez = z_error(n, z, sigma)
    if add:
        assert torch.equal(n, (x.detach()[some].float() + r.detach()[some].float()).to(dtype))
    close(y.detach()[some], want_y, ez * w.detach().double().abs() + 4 * U * (want_y.abs() + b.detach().double().abs()), "y")
    k = width / 256 + 16
    mh, mz = h.abs().mean(1, keepdim=True), (h * z).abs().mean(1, keepdim=True)
    emz = (h.abs() * ez).mean(1, keepdim=True) + k * U * mz
    edx = (8 * U * (h.abs() + mh + z.abs() * mz) + k * U * mh + ez * mz + z.abs() * emz) / sigma * 2
    if add:
        want_dx = want_dx + d.double()
        edx = edx + 4 * U * want_dx.abs()
    close(dx[some], want_dx, edx, "dx")
    # the sums over all rows, in parts of 64 bits
    want_dw, want_db, bound_w, bound_b = (torch.zeros(width, dtype=torch.float64, device="cuda") for _ in range(4))
    for a in range(0, rows, 4096):
        _, z, sigma, _, pw, pb, _ = reference(normalised[a : a + 4096], w.detach(), b.detach(), 1e-5, dy[a : a + 4096])
        g = dy[a : a + 4096].double().abs()
        want_dw += pw
        want_db += pb
        bound_w += (g * z_error(normalised[a : a + 4096], z, sigma)).sum(0) + rows * U * (g * z.abs()).sum(0)
        bound_b += rows * U * g.sum(0)
    close(dw, want_dw, bound_w, "dw")
    close(db, want_db, bound_b, "db")


def places(n, element_bytes):
    """Stretches of 64 elements at the ends and around what 32 bits wrap at."""
    marks = [0, n // 2, n - 64]
    for wrap in (1 << 31, 1 << 32):
        marks += [wrap - 32, wrap // element_bytes - 32]
    return sorted({m // 32 * 32 for m in marks if 0 <= m <= n - 64})


def test_adamw_32(ops):
    """1.1 G elements: byte offsets past 4 GiB in every list."""
    n, gen = 1_100_000_033, torch.Generator(device="cuda").manual_seed(1)
    p, g = randn((n,), torch.float32, gen, 0.5), randn((n,), torch.bfloat16, gen, 0.01)
    m, v = randn((n,), torch.float32, gen, 0.01), randn((n,), torch.float32, gen, 0.01).square_()
    c = torch.empty(n, dtype=torch.bfloat16, device="cuda")
    at = [slice(a, a + 64) for a in places(n, 4)]
    want = [formula(p[s], g[s], m[s], v[s], 7, **NUMBERS) for s in at]
    ops.adamw_step([p], [g], [m], [v], step=7, copies=[c], **NUMBERS)
    for s, (p2, m2, v2, ep, em, ev) in zip(at, want):
        for got, expect, bound in ((p, p2, ep), (m, m2, em), (v, v2, ev)):
            assert bool(((got[s].double() - expect).abs() <= bound).all()), s
        assert torch.equal(c[s], p[s].bfloat16())
    assert bool(c.isfinite().all())


def test_adamw_8(ops):
    """4.4 G elements: their numbers pass 32 bits, in the offsets and in what is hashed."""
    n, gen = (1 << 32) + 100_003, torch.Generator(device="cuda").manual_seed(2)
    p, g = (torch.zeros(n, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    codes = [torch.zeros(n, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2)]
    scales = [torch.zeros(-(-n // 32), dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu) for _ in range(2)]
    at = [slice(a, a + 64) for a in places(n, 2)] + [slice(n - n % 32 - 64, n - n % 32)]
    for s in at:
        p[s], g[s] = torch.randn(64, generator=gen, device="cuda") * 0.5, torch.randn(64, generator=gen, device="cuda") * 0.01
    before = [(p[s].clone(), g[s].clone()) for s in at]
    ops.adamw_step_8bit([p], [g], [codes[0]], [scales[0]], [codes[1]], [scales[1]], step=1, seed=5, **NUMBERS)
    for s, (old, grad) in zip(at, before):
        p2, m2, v2, ep, em, _ = formula(old, grad, torch.zeros(64, device="cuda"), torch.zeros(64, device="cuda"), 1, **NUMBERS)
        i = torch.arange(s.start, s.stop, device="cuda")
        word = mixed((i & 0xFFFFFFFF) + (i >> 32) * 0x632BE5AB + mixed(torch.tensor(5, device="cuda")) & 0xFFFFFFFF)
        blocks = slice(s.start // 32, s.stop // 32)
        for k, (x, half, power) in enumerate(((m2, word % 65536, 1), (v2.sqrt(), word // 65536, 2))):
            got = ops.dequantize_blocks(codes[k][s].clone(), scales[k][blocks].clone()).double()
            scale, low, high, share = neighbours(x, power)
            chance = (half.double() + 0.5) / 65536
            near = 2 * (em if power == 1 else 8 * U * x) / (scale * (high - low)) + 16 * U
            either = ((chance - share).abs() < near) | (share < near) | (share > 1 - near)
            assert bool(((got.abs() == torch.where(chance < share, high, low) * scale) | either).all()), (s, power)
        assert bool(((p[s].double() - p2).abs() <= p2.abs() * 2.0**-7 + ep).all())
    assert int(p.count_nonzero()) <= 64 * len(at)  # what had no gradient and no value has none now


def test_squared_norm(ops):
    n, gen = 2_200_000_011, torch.Generator(device="cuda").manual_seed(3)
    x = randn((n,), torch.bfloat16, gen, 0.3)
    want = sum(float(x[a : a + (1 << 27)].double().square().sum()) for a in range(0, n, 1 << 27))
    assert abs(float(ops.squared_norm([x])) - want) <= 64 * U * want
