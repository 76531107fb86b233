"""Tensors whose sign torch has put off (``x.conj().imag`` and its kin): their memory holds the negative of their values."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from odc_amd import ops

    assert torch.cuda.is_available(), "GPU test run without a GPU"
    return ops


def put_off(t):
    v = torch._neg_view(-t)
    assert v.is_neg() and torch.equal(v, t)
    return v


@pytest.mark.parametrize("width", [1, 8, 257, 4096])
def test_norms(ops, width):
    gen = torch.Generator(device="cuda").manual_seed(0)
    x, r, dy, dt = (torch.randn(9, width, generator=gen, device="cuda") for _ in range(4))
    w, b = (torch.randn(width, generator=gen, device="cuda") for _ in range(2))

    def results(x, r, w, b, dy, dt):
        leaves = [t.detach().requires_grad_() for t in (x, r, w, b)]
        assert [t.is_neg() for t in leaves] == [t.is_neg() for t in (x, r, w, b)]
        y, total = ops.add_layer_norm(leaves[0], leaves[1], width, leaves[2], leaves[3])
        grads = torch.autograd.grad((y, total), leaves, (dy, dt))
        return [y.detach(), total.detach(), ops.layer_norm(x, width, w, b), *grads]

    tensors = [x, r, w, b, dy, dt]
    want = results(*tensors)
    for k in range(6):
        got = results(*(put_off(t) if j == k else t for j, t in enumerate(tensors)))
        assert all(torch.equal(a, c) for a, c in zip(got, want)), k


def test_a_column_of_a_conjugate(ops):
    z = torch.randn(4, 1, dtype=torch.complex64, device="cuda").conj()
    _, total = ops.add_layer_norm(z.imag, torch.zeros(4, 1, device="cuda"), 1)
    assert torch.equal(total, z.imag.resolve_neg())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradients_of_a_step(ops, dtype):
    gen = torch.Generator(device="cuda").manual_seed(1)
    g = torch.randn(1000, generator=gen, device="cuda").to(dtype)
    out = []
    for grad in (g, put_off(g)):
        p, m, v = torch.ones(1000, device="cuda"), torch.zeros(1000, device="cuda"), torch.zeros(1000, device="cuda")
        ops.adamw_step([p], [grad], [m], [v], step=1, lr=0.1)
        w = torch.nn.Parameter(torch.ones(1000, device="cuda").to(dtype))
        w.grad = grad
        ops.AdamW([w], lr=0.1).step()
        out.append((p, m, v, w.detach()))
    assert all(torch.equal(a, b) for a, b in zip(*out))
    assert torch.equal(ops.squared_norm([g]), ops.squared_norm([put_off(g)]))


def test_what_is_written_is_no_such_view(ops):
    for place in (0, 2, 3):
        tensors = [torch.ones(8, device="cuda") for _ in range(4)]
        tensors[place] = put_off(tensors[place])
        with pytest.raises(ValueError, match="sign"):
            ops.adamw_step(*([t] for t in tensors), step=1, lr=0.1)
        assert all(bool((t == 1).all()) for t in tensors)
