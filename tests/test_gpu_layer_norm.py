"""odc_amd.ops.layer_norm / add_layer_norm / LayerNorm against the formula in 64 bits.

Bounds. u = 2^-24. The mean of a row is a sum of N terms of at most max|x|, made in N / 256 steps per thread or fewer
and a tree over the threads, so it is off by at most k u max|x| with k = N / 256 + 16; x - mean is off by that plus a
rounding, the variance's relative error is twice its terms'. With a = max|x| / sigma a value of z is therefore off by
less than k u (a + |z|) (1 + |z|) / 1, doubled here for the square root, the division and the products. A result in 16
bits is rounded once more (to 8 bits of bf16 or 11 of fp16: by 2^-8 or 2^-11 of its value at most)."""

import pytest
import torch

U = 2.0**-24
UNIT = {torch.float32: U, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
TINY = {torch.float32: 2.0**-149, torch.bfloat16: 2.0**-133, torch.float16: 2.0**-24}
pytestmark = pytest.mark.gpu

DTYPES = [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32),
          (torch.float16, torch.float16), (torch.float16, torch.float32)]
# one element, less than a vector, around wavefronts, vectors and the kernels' widths, odd ones, wide ones
WIDTHS = [1, 2, 3, 7, 8, 31, 33, 64, 65, 127, 129, 255, 256, 257, 500, 512, 513, 1001, 1024, 1025, 2047, 2048, 2056, 4096, 4099,
          8191, 8192, 8200, 14336, 16384, 16389, 20001, 33000]


@pytest.fixture(scope="module")
def ops():
    from odc_amd import ops

    assert torch.cuda.is_available(), "GPU test run without a GPU"
    return ops


def reference(x, w, b, eps, dy=None):
    """y, z, sigma (and the gradients) in 64 bits."""
    x = x.double()
    mean = x.mean(1, keepdim=True)
    sigma = ((x - mean).square().mean(1, keepdim=True) + eps).sqrt()
    z = (x - mean) / sigma
    y = z * (1 if w is None else w.double()) + (0 if b is None else b.double())
    if dy is None:
        return y, z, sigma
    dy = dy.double()
    h = dy * (1 if w is None else w.double())
    dx = (h - h.mean(1, keepdim=True) - z * (h * z).mean(1, keepdim=True)) / sigma
    return y, z, sigma, dx, (dy * z).sum(0), dy.sum(0), h


def close(got, want, slack, what):
    bound = slack + UNIT[got.dtype] * want.abs() + TINY[got.dtype]
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), f"{what}: off by {float((off / bound).max()):.3g} of the bound"


def z_error(x, z, sigma):
    k = x.shape[1] / 256 + 16
    a = x.double().abs().amax(1, keepdim=True) / sigma
    return 2 * k * U * (a + z.abs()) * (1 + z.abs())


def check(ops, rows, width, dtype, wdtype, gen, add=False, weight=True, bias=True, pad=0, offset=0.3, eps=1e-5, backward=True):
    def randn(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    def slice_of_wider():
        wide = (randn(rows, width + pad) * 1.5 + offset).to(dtype)
        return wide[:, pad // 2 : pad // 2 + width].requires_grad_(backward)

    x = slice_of_wider()
    r = slice_of_wider() if add else None
    w = (1 + 0.2 * randn(width)).to(wdtype).requires_grad_(backward) if weight else None
    b = (0.2 * randn(width)).to(wdtype).requires_grad_(backward) if bias else None
    if add:
        y, total = ops.add_layer_norm(x, r, (width,), w, b, eps)
        assert torch.equal(total, (x.detach().float() + r.detach().float()).to(dtype))  # one rounding of the exact or fp32 sum
        normalised = total.detach()
    else:
        y = ops.layer_norm(x, (width,), w, b, eps)
        normalised = x.detach()
    assert y.shape == x.shape and y.dtype == dtype and y.is_contiguous()
    dy, dtotal = (randn(rows, width) * 0.1).to(dtype), (randn(rows, width) * 0.1).to(dtype)
    want_y, z, sigma, want_dx, want_dw, want_db, h = reference(normalised, None if w is None else w.detach(), None if b is None else b.detach(), eps, dy)
    ez = z_error(normalised, z, sigma)
    wabs = 1 if w is None else w.detach().double().abs()
    babs = 0 if b is None else b.detach().double().abs()
    close(y.detach(), want_y, ez * wabs + 4 * U * (z.abs() * wabs + babs), "y")
    if not backward:
        return
    inputs = [t for t in (x, r, w, b) if t is not None]
    grads = torch.autograd.grad((y, total) if add else y, inputs, (dy, dtotal) if add else dy)
    grads = dict(zip([n for n, t in zip("xrwb", (x, r, w, b)) if t is not None], grads))
    # dx is made of h, its mean and z's mean with it: sums as above, with z's error in them
    k = width / 256 + 16
    mh, mz = h.abs().mean(1, keepdim=True), (h * z).abs().mean(1, keepdim=True)
    emz = (h.abs() * ez).mean(1, keepdim=True) + k * U * mz
    edx = (8 * U * (h.abs() + mh + z.abs() * mz) + k * U * mh + ez * mz + z.abs() * emz) / sigma * 2
    if add:
        want_dx = want_dx + dtotal.double()
        edx = edx + 4 * U * want_dx.abs()
        assert torch.equal(grads["r"], grads["x"])
    close(grads["x"], want_dx, edx, "dx")
    kr = rows + 16  # terms of a column's sum, at most one rounding each
    if weight:
        close(grads["w"], want_dw, ((dy.double().abs() * ez).sum(0) + kr * U * (dy.double() * z).abs().sum(0)), "dw")
    if bias:
        close(grads["b"], want_db, kr * U * dy.double().abs().sum(0), "db")


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("dtype,wdtype", DTYPES)
def test_widths(ops, width, dtype, wdtype):
    gen = torch.Generator(device="cuda").manual_seed(width)
    for rows in (1, 5, 131):
        check(ops, rows, width, dtype, wdtype, gen, add=rows == 5)


@pytest.mark.parametrize("rows", [1, 2, 3, 4, 63, 64, 255, 256, 257, 1023, 4097])
@pytest.mark.parametrize("width", [8, 96, 768, 2500])
def test_rows(ops, rows, width):
    gen = torch.Generator(device="cuda").manual_seed(rows)
    check(ops, rows, width, torch.bfloat16, torch.float32, gen)
    check(ops, rows, width, torch.float32, torch.float32, gen, add=True)


@pytest.mark.parametrize("pad", [1, 2, 5, 8, 64, 101])
@pytest.mark.parametrize("width", [33, 256, 1000, 4096, 17000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_of_a_wider_tensor(ops, pad, width, dtype):
    gen = torch.Generator(device="cuda").manual_seed(pad)
    check(ops, 37, width, dtype, torch.float32, gen, add=pad % 2 == 0, pad=pad)


@pytest.mark.parametrize("weight,bias", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("add", [False, True])
@pytest.mark.parametrize("width", [64, 3001, 20000])
def test_without_weight_or_bias(ops, weight, bias, add, width):
    gen = torch.Generator(device="cuda").manual_seed(3)
    check(ops, 21, width, torch.bfloat16, torch.float32, gen, add=add, weight=weight, bias=bias)
    check(ops, 21, width, torch.float32, torch.float32, gen, add=add, weight=weight, bias=bias)


def test_forward_only(ops):
    gen = torch.Generator(device="cuda").manual_seed(4)
    for width in (3, 256, 4096, 18001):
        check(ops, 9, width, torch.float16, torch.float16, gen, add=True, backward=False)


def test_a_large_mean_does_not_cost_the_variance(ops):
    gen = torch.Generator(device="cuda").manual_seed(5)
    for width in (100, 4096, 20000):
        check(ops, 6, width, torch.float32, torch.float32, gen, offset=3000.0)


def test_every_derivative_against_differences(ops):
    """Along random directions, against central differences of the formula in 64 bits (their own error: 1e-9)."""
    gen = torch.Generator(device="cuda").manual_seed(6)
    for rows, width in ((3, 5), (17, 130), (40, 2049)):
        x, r, dy, dt = (torch.randn(rows, width, generator=gen, device="cuda") for _ in range(4))
        w, b = (torch.randn(width, generator=gen, device="cuda") for _ in range(2))
        leaves = [t.requires_grad_() for t in (x, r, w, b)]
        y, total = ops.add_layer_norm(x, r, width, w, b)
        grads = torch.autograd.grad((y, total), leaves, (dy, dt))

        def loss(x, r, w, b):
            t = x + r
            return float((reference(t, w, b, 1e-5)[0] * dy.double()).sum() + (t * dt.double()).sum())

        values = [t.detach().double() for t in leaves]
        for k, g in enumerate(grads):
            d = torch.randn(g.shape, generator=gen, device="cuda").double()
            h = 1e-5
            up, down = (loss(*(v + s * h * d if j == k else v for j, v in enumerate(values))) for s in (1, -1))
            want, terms = (up - down) / (2 * h), float((g.double() * d).abs().sum())
            assert abs(float((g.double() * d).sum()) - want) < 1e-4 * terms + 1e-5, (rows, width, k)


def test_leading_dimensions_and_layouts(ops):
    gen = torch.Generator(device="cuda").manual_seed(7)
    base = torch.randn(4, 6, 5, 96, generator=gen, device="cuda")
    w, b = torch.randn(96, generator=gen, device="cuda"), torch.randn(96, generator=gen, device="cuda")
    views = [base, base[:, 1:4], base[::2], base.transpose(1, 2), base.permute(3, 1, 0, 2).contiguous().permute(2, 1, 3, 0),
             base[0, 0, 0], base[:, :1, :1].expand(4, 6, 5, 96), base[..., 3:35][..., :32]]
    for v in views:
        n = v.shape[-1]
        want = reference(v.reshape(-1, n), w[:n], b[:n], 1e-5)[0].view(v.shape)
        got = ops.layer_norm(v, (n,), w[:n], b[:n])
        assert got.shape == v.shape and float((got.double() - want).abs().max()) < 1e-5
    # several normalised dimensions
    v = base[:, ::2]
    w2, b2 = torch.randn(5, 96, generator=gen, device="cuda"), torch.randn(5, 96, generator=gen, device="cuda")
    want = reference(v.reshape(-1, 480), w2.view(-1), b2.view(-1), 1e-5)[0].view(v.shape)
    assert float((ops.layer_norm(v, (5, 96), w2, b2).double() - want).abs().max()) < 1e-5
    # gradients of any layout, broadcast ones among them
    for dy in (torch.ones((), device="cuda").expand(4, 6, 5, 96), torch.randn(4, 5, 6, 96, generator=gen, device="cuda").transpose(1, 2),
               torch.randn(4, 6, 5, 100, generator=gen, device="cuda")[..., 2:98]):
        x = base.clone().requires_grad_()
        dx, = torch.autograd.grad(ops.layer_norm(x, 96, w, b), x, dy)
        want = reference(x.detach().view(-1, 96), w, b, 1e-5, dy.reshape(-1, 96))[3].view(dx.shape)
        assert dx.shape == x.shape and float((dx.double() - want).abs().max()) < 1e-5


def test_gradients_that_are_not_asked_for(ops):
    gen = torch.Generator(device="cuda").manual_seed(8)
    x, r = (torch.randn(33, 200, generator=gen, device="cuda") for _ in range(2))
    w, b = (torch.randn(200, generator=gen, device="cuda") for _ in range(2))
    dy = torch.randn(33, 200, generator=gen, device="cuda")
    _, _, _, dx, dw, db, _ = reference(x, w, b, 1e-5, dy)
    for wants in ("x", "w", "b", "xw", "wb"):
        named = {n: t.clone().requires_grad_(n in wants) for n, t in (("x", x), ("w", w), ("b", b))}
        y = ops.layer_norm(named["x"], 200, named["w"], named["b"])
        for n, g in zip(wants, torch.autograd.grad(y, [named[n] for n in wants], dy)):
            want = {"x": dx, "w": dw, "b": db}[n]
            assert float((g.double() - want).abs().max()) < 1e-4, (wants, n)
    # of the two results only one is used
    x1, r1, w1 = x.clone().requires_grad_(), r.clone().requires_grad_(), w.clone().requires_grad_()
    _, total = ops.add_layer_norm(x1, r1, 200, w1, b)
    gx, gr, gw = torch.autograd.grad(total, (x1, r1, w1), dy, allow_unused=True)
    assert torch.equal(gx, dy) and torch.equal(gr, dy) and gw is None
    y, _ = ops.add_layer_norm(x1, r1, 200, w1, b)
    gx, gr = torch.autograd.grad(y, (x1, r1), dy)
    want = reference((x + r), w, b, 1e-5, dy)[3]
    assert torch.equal(gx, gr) and float((gx.double() - want).abs().max()) < 1e-4
    with pytest.raises(RuntimeError, match="second derivative"):
        y = ops.layer_norm(x1, 200, w1, b)
        g, = torch.autograd.grad(y, x1, dy, create_graph=True)
        torch.autograd.grad(g.sum(), x1)


def test_rows_do_not_see_each_other(ops):
    """Infinities, NaN and rows of one value: what a row holds stays in it."""
    gen = torch.Generator(device="cuda").manual_seed(9)
    for rows, width in ((40, 24), (40, 500), (9, 4096), (5, 17000)):
        x = torch.randn(rows, width, generator=gen, device="cuda")
        x[1, 0], x[2, width - 1], x[3] = float("nan"), float("inf"), 7.5
        x[4] = 3e38
        clean = x.clone()
        clean[1:5] = torch.randn(4, width, generator=gen, device="cuda")[: len(clean[1:5])]
        dy = torch.randn(rows, width, generator=gen, device="cuda")
        got, other = ops.layer_norm(x, width), ops.layer_norm(clean, width)
        keep = [i for i in range(rows) if i not in (1, 2, 3, 4)]
        assert torch.equal(got[keep], other[keep])
        assert bool(got[1].isnan().all()) and bool(got[2].isnan().all())
        assert bool((got[3] == 0).all())  # variance 0: eps alone is divided by
        a, c = x.clone().requires_grad_(), clean.clone().requires_grad_()
        da, = torch.autograd.grad(ops.layer_norm(a, width), a, dy)
        dc, = torch.autograd.grad(ops.layer_norm(c, width), c, dy)
        assert torch.equal(da[keep], dc[keep])


def test_empty(ops):
    w, b = torch.ones(16, device="cuda", requires_grad=True), torch.ones(16, device="cuda", requires_grad=True)
    x = torch.empty(0, 16, device="cuda", requires_grad=True)
    y = ops.layer_norm(x, 16, w, b)
    assert y.shape == (0, 16)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty(0, 16, device="cuda"))
    assert dx.shape == (0, 16) and not dw.any() and not db.any()
    y, total = ops.add_layer_norm(x, x, 16, w, b)
    assert y.shape == total.shape == (0, 16)


def test_the_same_inputs_give_the_same_bits(ops):
    gen = torch.Generator(device="cuda").manual_seed(10)
    for rows, width in ((2048, 256), (777, 1001), (300, 9000)):
        x = torch.randn(rows, width, generator=gen, device="cuda").bfloat16().requires_grad_()
        w = torch.randn(width, generator=gen, device="cuda").requires_grad_()
        dy = torch.randn(rows, width, generator=gen, device="cuda").bfloat16()
        runs = []
        for _ in range(3):
            y = ops.layer_norm(x, width, w)
            runs.append((y, *torch.autograd.grad(y, (x, w), dy)))
        for run in runs[1:]:
            assert all(torch.equal(a, b) for a, b in zip(run, runs[0]))


def test_on_another_stream_and_in_a_graph(ops):
    gen = torch.Generator(device="cuda").manual_seed(11)
    x = torch.randn(600, 768, generator=gen, device="cuda").requires_grad_()
    w, b = (torch.randn(768, generator=gen, device="cuda").requires_grad_() for _ in range(2))
    dy = torch.randn(600, 768, generator=gen, device="cuda")

    def step():
        # (no autograd graph outlives the call: its nodes of the leaves would belong to this stream, and a backward pass
        # that is captured later on another one would make the two wait for each other)
        y = ops.layer_norm(x, 768, w, b)
        grads = torch.autograd.grad(y, (x, w, b), dy)
        return (y.detach(), *grads)

    eager = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(other, eager))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for _ in range(3):
        for t in captured:
            t.fill_(7)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(captured, eager))
        assert torch.equal(step()[1], eager[1])


def test_module(ops):
    torch.manual_seed(0)
    ours, theirs = ops.LayerNorm(160).cuda(), torch.nn.LayerNorm(160).cuda()
    with torch.no_grad():
        theirs.weight.normal_()
        theirs.bias.normal_()
    ours.load_state_dict(theirs.state_dict())
    x, r = torch.randn(3, 7, 160, device="cuda"), torch.randn(3, 7, 160, device="cuda")
    assert torch.allclose(ours(x), theirs(x), atol=1e-5)
    y, total = ours(x, r)
    assert torch.allclose(y, theirs(x + r), atol=1e-5) and torch.equal(total, x + r)
    plain = ops.LayerNorm(160, elementwise_affine=False).cuda()
    assert torch.allclose(plain(x), torch.nn.functional.layer_norm(x, (160,)), atol=1e-5)


def test_refusals(ops):
    x, w = torch.randn(4, 32, device="cuda"), torch.ones(32, device="cuda")
    with pytest.raises(TypeError, match="GPU"):
        ops.layer_norm(x.cpu(), 32)
    with pytest.raises(TypeError, match="bf16, fp16 or fp32"):
        ops.layer_norm(x.double(), 32)
    with pytest.raises(ValueError, match="normalized_shape"):
        ops.layer_norm(x, 31)
    with pytest.raises(ValueError, match="normalized_shape"):
        ops.layer_norm(x, (2, 4, 32))
    with pytest.raises(ValueError, match="normalized_shape"):
        ops.layer_norm(x, ())
    with pytest.raises(ValueError, match="weight"):
        ops.layer_norm(x, 32, w[:31])
    with pytest.raises(TypeError, match="weight"):
        ops.layer_norm(x, 32, w.half())
    with pytest.raises(TypeError, match="different dtypes"):
        ops.layer_norm(x.half(), 32, w, w.half())
    with pytest.raises(TypeError, match="GPU"):
        ops.layer_norm(x, 32, w.cpu())
    with pytest.raises(ValueError, match="residual"):
        ops.add_layer_norm(x, x[:3], 32)
    with pytest.raises(TypeError, match="residual"):
        ops.add_layer_norm(x, x.half(), 32)
    with pytest.raises(TypeError, match="residual"):
        ops.add_layer_norm(x, x.cpu(), 32)
    with pytest.raises(ValueError, match="eps"):
        ops.layer_norm(x, 32, eps=-1.0)
    with pytest.raises(TypeError, match="torch.Tensor"):
        ops.layer_norm([1.0], 1)
