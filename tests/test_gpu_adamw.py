"""odc_amd.ops.adamw_step / adamw_step_8bit / squared_norm / dequantize_blocks / AdamW against the formulas in 64 bits.

Bounds. u = 2^-24. m and v are two products and a sum, each rounded once, of factors that are rounded to fp32: 4 u of
|beta m| + |(1 - beta) g| (g itself 2 u where it is scaled). The root, its scaling, the division and the step size add
at most 16 u of the update, and the decay's product and the last difference 2 u of |p|. Where a result has 16 bits
it is rounded once more (to 8 bits of bf16 or 11 of fp16: by 2^-8 or 2^-11 of its value at most)."""

import copy
import math

import pytest
import torch

U = 2.0**-24
UNIT = {torch.float32: 0.0, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
pytestmark = pytest.mark.gpu

NUMBERS = dict(lr=3e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1)
# one element, around vectors, blocks, tiles; more tensors than one launch takes; empty ones between
SIZES = {"one": [1], "few": [3, 1, 31, 32, 33, 64, 65], "tiles": [1023, 1024, 1025, 4096, 8191, 12289, 40003],
         "many": [1 + 37 * k % 700 for k in range(130)], "empty": [0, 5, 0, 0, 2049, 0]}


@pytest.fixture(scope="module")
def ops():
    from odc_amd import ops

    assert torch.cuda.is_available(), "GPU test run without a GPU"
    return ops


def make(sizes, dtype, scale, gen, shift=0):
    """Tensors that start ``shift`` elements behind an allocation's beginning."""
    out = []
    for n in sizes:
        t = torch.empty(n + shift, dtype=dtype, device="cuda")[shift:]
        out.append(t.copy_(torch.randn(n, generator=gen, device="cuda") * scale))
    return out


def formula(p, g, m, v, t, lr, betas, eps, weight_decay, factor=1.0):
    """The step in 64 bits: p, m, v, and the bounds of what fp32 makes of them."""
    p, g, m, v = p.double(), g.double() * factor, m.double(), v.double()
    b1, b2 = betas
    m2, v2 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    update = lr / (1 - b1**t) * m2 / (v2.sqrt() / math.sqrt(1 - b2**t) + eps)
    em = 6 * U * ((b1 * m).abs() + ((1 - b1) * g).abs())
    ev = 8 * U * v2
    eu = update.abs() * 24 * U + lr / (1 - b1**t) * em / (v2.sqrt() / math.sqrt(1 - b2**t) + eps)
    p2 = p * (1 - lr * weight_decay) - update
    return p2, m2, v2, eu + 4 * U * p.abs() + 2.0**-149, em + 2.0**-149, ev + 2.0**-149


def close(got, want, slack, what):
    bound = slack + UNIT[got.dtype] * want.abs()
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), f"{what}: off by {float((off / bound).max()):.3g} of the bound"


@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("param,grad,copied", [
    (torch.float32, torch.float32, None), (torch.float32, torch.bfloat16, torch.bfloat16), (torch.float32, torch.float16, torch.float16),
    (torch.bfloat16, torch.bfloat16, None), (torch.bfloat16, torch.float32, None), (torch.bfloat16, torch.float16, None)])
@pytest.mark.parametrize("shift", [0, 1, 3])
def test_steps_32(ops, sizes, param, grad, copied, shift):
    gen = torch.Generator(device="cuda").manual_seed(1)
    n = SIZES[sizes]
    ps, gs = make(n, param, 0.5, gen, shift), make(n, grad, 0.01, gen, shift)
    ms, vs = make(n, torch.float32, 0, gen, shift), make(n, torch.float32, 0, gen, shift)
    cs = make(n, copied, 0, gen, shift) if copied else None
    for t in (1, 2, 3):
        want = [formula(p, g, m, v, t, **NUMBERS) for p, g, m, v in zip(ps, gs, ms, vs)]
        ops.adamw_step(ps, gs, ms, vs, step=t, copies=cs, **NUMBERS)
        for k, (p2, m2, v2, ep, em, ev) in enumerate(want):
            close(ps[k], p2, ep, f"param {k}")
            close(ms[k], m2, em, f"m {k}")
            close(vs[k], v2, ev, f"v {k}")
            if copied:
                assert torch.equal(cs[k], ps[k].to(copied))
        gs = make(n, grad, 0.01, gen, shift)


def test_what_lies_around_the_tensors_stays(ops):
    gen = torch.Generator(device="cuda").manual_seed(2)
    for dtype in (torch.float32, torch.bfloat16):
        for n in (1, 5, 31, 1000, 4097):
            flats = [torch.full((n + 200,), 3.0, dtype=d, device="cuda") for d in (dtype, torch.float32, torch.float32)]
            g = torch.randn(n, generator=gen, device="cuda")
            p, m, v = (f[100 : 100 + n] for f in flats)
            ops.adamw_step([p], [g], [m], [v], step=5, **NUMBERS)
            for f in flats:
                assert bool((f[:100] == 3).all()) and bool((f[100 + n :] == 3).all())
                # (a step of 3e-3 is less than half a unit of 3 in bf16)
                assert f.dtype == torch.bfloat16 or not bool((f[100 : 100 + n] == 3).any())


@pytest.mark.parametrize("scale", [1.0, 0.125])
@pytest.mark.parametrize("max_norm", [0.5, 1e6, 0.0])
def test_clipping(ops, scale, max_norm):
    gen = torch.Generator(device="cuda").manual_seed(3)
    n = SIZES["tiles"]
    ps, gs = make(n, torch.float32, 0.5, gen), make(n, torch.float32, 0.3, gen)
    ms, vs = make(n, torch.float32, 0.1, gen), [v.abs_() for v in make(n, torch.float32, 0.1, gen)]
    norm = math.sqrt(sum(float(g.double().square().sum()) for g in gs)) * scale
    factor = scale * min(1.0, max_norm / (norm + 1e-6))
    want = [formula(p, g, m, v, 9, factor=factor, **NUMBERS) for p, g, m, v in zip(ps, gs, ms, vs)]
    ops.adamw_step(ps, gs, ms, vs, step=9, grad_scale=scale, squared_norm=ops.squared_norm(gs), max_norm=max_norm, **NUMBERS)
    for k, (p2, m2, v2, ep, em, ev) in enumerate(want):
        close(ps[k], p2, 2 * ep, f"param {k}")  # the factor has four roundings more
        close(ms[k], m2, 2 * em, f"m {k}")
        close(vs[k], v2, 2 * ev, f"v {k}")


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_gradient_that_is_not_finite(ops, bad):
    """Without clipping it reaches its own element alone; a norm that is not a number reaches all of them."""
    gen = torch.Generator(device="cuda").manual_seed(4)
    for eight in (False, True):
        p, g = make([300], torch.float32, 0.5, gen)[0], make([300], torch.float32, 0.1, gen)[0]
        g[77] = bad
        twin_g = g.clone()
        twin_g[77] = 0
        results = []
        for grad in (g, twin_g):
            q, states = p.clone(), new_states(ops, 300, eight)
            call(ops, [q], [grad], [states], 1)
            results.append((q, *values(ops, states)))
        keep = torch.arange(300, device="cuda") != 77
        for a, b in zip(*results):
            if not eight or a is results[0][0]:
                assert torch.equal(a[keep], b[keep])
            assert bool(a[77].isnan() | a[77].isinf())
        if eight:  # its block keeps a scale made of the others (which differs from the twin's by nothing here)
            assert bool(results[0][1][keep].isfinite().all()) and bool(results[0][2][keep].isfinite().all())
    if bad != bad:
        q, m, v = p.clone(), torch.zeros_like(p), torch.zeros_like(p)
        ops.adamw_step([q], [g], [m], [v], step=1, squared_norm=ops.squared_norm([g]), max_norm=1.0, **NUMBERS)
        assert bool(q.isnan().all())


# ---- 8 bits -----------------------------------------------------------------------------------------
def new_states(ops, n, eight=True):
    if not eight:
        return [torch.zeros(n, device="cuda") for _ in range(2)]
    sizes, kinds = (n, -(-n // 32)) * 2, (torch.float8_e4m3fn, torch.float8_e8m0fnu) * 2
    return [torch.zeros(s, dtype=torch.uint8, device="cuda").view(k) for s, k in zip(sizes, kinds)]


def call(ops, ps, gs, states, t, seed=None, **more):
    lists = [list(x) for x in zip(*states)]
    if len(lists) == 2:
        ops.adamw_step(ps, gs, *lists, step=t, **{**NUMBERS, **more})
    else:
        ops.adamw_step_8bit(ps, gs, *lists, step=t, seed=t if seed is None else seed, **{**NUMBERS, **more})


def values(ops, states):
    """m and v (or m and the root) in fp32."""
    if len(states) == 2:
        return [s.clone() for s in states]
    return [ops.dequantize_blocks(states[0], states[1]), ops.dequantize_blocks(states[2], states[3])]


def mixed(x):
    x = ((x ^ (x >> 16)) * 0xB7E15163) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0x9E3779B1) & 0xFFFFFFFF
    return x ^ (x >> 16)


def words(n, k, seed):
    return mixed(torch.arange(n, device="cuda") + mixed(torch.tensor((seed + k * 0x9E3779B1) & 0xFFFFFFFF, device="cuda")) & 0xFFFFFFFF)


def neighbours(x, power):
    """For every value of x: its block's scale, the codes' values below and above, and the share of the way."""
    n = x.numel()
    blocks = torch.nn.functional.pad(x.abs(), (0, -n % 32)).view(-1, 32)
    k = torch.ceil(torch.log2(blocks.amax(1).clamp(min=1e-200) / 448)).clamp(min=-117)
    scale = torch.exp2(k).repeat_interleave(32)[:n]
    a = x.abs() / scale
    if power == 2:
        a = torch.where(a > 0, a.clamp(min=2.0**-9), a)
    ulp = torch.exp2(torch.floor(torch.log2(a.clamp(min=2.0**-6))) - 3)
    low = torch.floor(a / ulp) * ulp
    return scale, low, low + ulp, (a**power - low**power) / ((low + ulp) ** power - low**power)


def check_stored(got, want, slack, half, power, what):
    """Every stored value is the neighbour that its 16 random bits choose. What fp32 is off by (``slack``), as a share of
    the distance of the two codes, may make the other one of it where the chance is as near to the share as that; the
    comparison itself has a few roundings. Between squares the share of the way changes by less than twice as much."""
    scale, low, high, share = neighbours(want, power)
    chance = (half.double() + 0.5) / 65536
    chosen = torch.where(chance < share, high, low) * scale
    near = 2 * slack / (scale * (high - low)) + 16 * U
    either = (chance - share).abs() < near
    edge = (share < near) | (share > 1 - near)  # the value itself may have crossed a code
    off = (got.abs().double() - chosen).abs()
    wrong = off > 0
    assert not bool((wrong & ~either & ~edge).any()), f"{what}: {int((wrong & ~either & ~edge).sum())} of {got.numel()} are another code"
    assert bool((off <= 1.01 * (high - low) * scale)[wrong].all()), what
    if power == 1:  # (a sum that cancels to less than its error may have either sign)
        assert bool((torch.signbit(got) == torch.signbit(want))[want.abs() > slack].all()), what
    assert int(wrong.sum()) <= 2 + got.numel() // 500, what


@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("param,grad,copied", [
    (torch.float32, torch.float32, None), (torch.float32, torch.bfloat16, torch.bfloat16), (torch.float32, torch.float16, torch.float16),
    (torch.bfloat16, torch.bfloat16, None), (torch.bfloat16, torch.float32, None)])
@pytest.mark.parametrize("shift", [0, 1])
def test_steps_8(ops, sizes, param, grad, copied, shift):
    gen = torch.Generator(device="cuda").manual_seed(5)
    n = SIZES[sizes]
    ps = make(n, param, 0.5, gen, shift)
    states = [new_states(ops, size) for size in n]
    if shift:  # states that begin at no boundary
        for s in states:
            for j in range(4):
                s[j] = torch.cat([torch.zeros(shift, dtype=torch.uint8, device="cuda"), s[j].view(torch.uint8)])[shift:].view(s[j].dtype)
    cs = make(n, copied, 0, gen, shift) if copied else None
    for t in (1, 2, 3):
        gs = make(n, grad, 0.01, gen, shift)
        for g in gs:
            g *= torch.exp2(torch.randint(-6, 7, g.shape, generator=gen, device="cuda").float()).to(grad)
        before = [(p.clone(), *values(ops, s)) for p, s in zip(ps, states)]
        call(ops, ps, gs, states, t, seed=77 + t, copies=cs)
        for k, size in enumerate(n):
            p, m, root = before[k]
            p2, m2, v2, ep, em, ev = formula(p, gs[k], m, root.double() ** 2, t, **NUMBERS)
            word = words(size, k, 77 + t)
            if param == torch.bfloat16:
                ulp = torch.exp2(torch.floor(torch.log2(p2.abs().clamp(min=2.0**-126))) - 7)
                share, chance = p2.abs() / ulp % 1, (mixed(word ^ 0x5BF03635) % 65536).double() / 65536
                chosen = torch.sign(p2) * (p2.abs() / ulp).floor() * ulp + torch.sign(p2) * torch.where(chance + share >= 1, ulp, 0)
                slack = 2 * ep / ulp + 2.0**-15
                near = ((chance + share - 1).abs() < slack) | (share < slack) | (share > 1 - slack)
                assert not bool(((ps[k].double() != chosen) & ~near).any()), f"param {k}"
                assert bool(((ps[k].double() - p2).abs() <= 1.01 * ulp + ep).all()), f"param {k}"
            else:
                close(ps[k], p2, ep + 4 * U * p2.abs(), f"param {k}")
            if copied:
                assert torch.equal(cs[k], ps[k].to(copied))
            m_now, root_now = values(ops, states[k])
            check_stored(m_now, m2, em, word % 65536, 1, f"m {k}")
            check_stored(root_now, v2.sqrt(), 8 * U * v2.sqrt(), word // 65536, 2, f"root {k}")


def test_what_lies_around_states_in_8_bits_stays(ops):
    gen = torch.Generator(device="cuda").manual_seed(6)
    for n in (1, 5, 31, 33, 1000, 4097):
        blocks = -(-n // 32)
        flats = [torch.full((size + 200,), 0x30, dtype=torch.uint8, device="cuda") for size in (n, blocks) * 2]
        p = torch.randn(n + 200, generator=gen, device="cuda")
        kept = p.clone()
        g = torch.randn(n, generator=gen, device="cuda")
        kinds = (torch.float8_e4m3fn, torch.float8_e8m0fnu) * 2
        states = [f[100 : 100 + size].view(kind) for f, size, kind in zip(flats, (n, blocks) * 2, kinds)]
        for s in states:
            s.view(torch.uint8).zero_()
        call(ops, [p[100 : 100 + n]], [g], [states], 1)
        for f, size in zip(flats, (n, blocks) * 2):
            assert bool((f[:100] == 0x30).all()) and bool((f[100 + size :] == 0x30).all())
        assert torch.equal(p[:100], kept[:100]) and torch.equal(p[100 + n :], kept[100 + n :])


def test_expectations_are_kept(ops):
    """Over seeds the mean of what is stored is m, and the mean of the square of the stored root is v: 4000 draws of a
    value between two codes have a standard error of at most half their distance / sqrt(4000); 5 of them are allowed."""
    gen = torch.Generator(device="cuda").manual_seed(7)
    draws, n = 4000, 96
    g = make([n], torch.float32, 0.02, gen)[0] * torch.exp2(torch.randint(-4, 5, (n,), generator=gen, device="cuda").float())
    p = torch.zeros(n, device="cuda")
    sums = torch.zeros(2, n, dtype=torch.float64, device="cuda")
    for seed in range(draws):
        states = new_states(ops, n)
        call(ops, [p.clone()], [g], [states], 1, seed=seed * 7919 + 1)
        m, root = values(ops, states)
        sums += torch.stack([m.double(), root.double() ** 2])
    _, m2, v2, *_ = formula(p, g, torch.zeros_like(p), torch.zeros_like(p), 1, **NUMBERS)
    for got, want, power in zip(sums / draws, (m2, v2), (1, 2)):
        scale, low, high, _ = neighbours(want if power == 1 else want.sqrt(), power)
        distance = (high**power - low**power) * scale**power
        small = want.abs() < (2.0**-9 * scale) ** power if power == 2 else torch.zeros_like(want, dtype=torch.bool)
        assert bool((((got - want).abs() <= 5 * 0.5 * distance / math.sqrt(draws) + 1e-12)[~small]).all())


def test_an_average_of_8_bits_moves(ops):
    """v starts at what large gradients left and decays to what small ones give: its mean over many elements follows
    the 64 bit average. Rounded to the nearest code it would stay where it was for ever."""
    n, t = 1 << 15, 1
    gen = torch.Generator(device="cuda").manual_seed(8)
    p, states = torch.zeros(n, device="cuda"), new_states(ops, n)
    v, m = 0.0, 0.0
    for scale in (1.0, 0.25):
        for _ in range(300):
            g = torch.full((n,), scale, device="cuda")
            call(ops, [p], [g], [states], t, lr=0.0, betas=(0.9, 0.99))
            v, m, t = 0.99 * v + 0.01 * scale**2, 0.9 * m + 0.1 * scale, t + 1
        got_m, got_root = values(ops, states)
        assert abs(float((got_root.double() ** 2).mean()) / v - 1) < 0.02, scale
        assert abs(float(got_m.double().mean()) / m - 1) < 0.02, scale
    assert v < 0.15  # it did move


def test_a_small_second_moment_is_not_stored_as_zero(ops):
    g = torch.zeros(64, device="cuda")
    g[0], g[1], g[2:32] = 1.0, 1e-9, 1e-30
    states = new_states(ops, 64)
    call(ops, [torch.zeros(64, device="cuda")], [g], [states], 1)
    m, root = values(ops, states)
    assert bool((root[:2] > 0).all()) and bool((root[32:] == 0).all()) and bool((m[32:] == 0).all())
    # 1e-30 squared is no fp32 number: its v is zero, and so is its root
    assert bool((root[2:32] == 0).all())


def test_seeds(ops):
    gen = torch.Generator(device="cuda").manual_seed(9)
    g = make([5000, 300], torch.float32, 0.02, gen)
    out = []
    for seed in (1, 1, 2, 2**32 + 1, -1):
        states = [new_states(ops, n) for n in (5000, 300)]
        call(ops, [torch.zeros(n, device="cuda") for n in (5000, 300)], g, states, 1, seed=seed)
        out.append([s.view(torch.uint8).clone() for one in states for s in one])
    same = [all(torch.equal(a, b) for a, b in zip(o, out[0])) for o in out]
    assert same == [True, True, False, True, False]


def test_stochastic_parameters(ops):
    """bf16 parameters with a seed: the mean moves by what a step adds up to, which the nearest value would lose."""
    n = 1 << 16
    for seed, moves in ((None, False), (3, True)):
        p = torch.ones(n, dtype=torch.bfloat16, device="cuda")
        g, m, v = torch.ones(n, device="cuda"), torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
        for t in range(1, 11):
            ops.adamw_step([p], [g], [m], [v], step=t, lr=1e-4, seed=None if seed is None else seed + t)
        mean = float(p.double().mean())
        assert (abs(mean - (1 - 1e-3)) < 1e-4) if moves else mean == 1.0


# ---- squared norm -----------------------------------------------------------------------------------
@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shift", [0, 1])
def test_squared_norm(ops, sizes, dtype, shift):
    gen = torch.Generator(device="cuda").manual_seed(10)
    ts = make(SIZES[sizes], dtype, 0.3, gen, shift)
    want = sum(float(t.double().square().sum()) for t in ts)
    got = ops.squared_norm(ts)
    assert got.shape == () and got.dtype == torch.float32
    # a thread adds up to 8192 / 256 squares per tile, rounded each, over a few tiles here: 64 u in all
    assert abs(float(got) - want) <= 64 * U * want
    assert torch.equal(got, ops.squared_norm(ts))


def test_squared_norm_of_much_and_of_little(ops):
    gen = torch.Generator(device="cuda").manual_seed(11)
    big = torch.randn(100_000_007, generator=gen, device="cuda")
    want = float(big.double().square().sum())
    # 12208 tiles over 2048 workgroups: 6 tiles of 32 squares for a thread
    assert abs(float(ops.squared_norm([big])) - want) <= 256 * U * want
    many = [big[k * 50 : k * 50 + 49] for k in range(1000)]  # seven launches
    want = sum(float(t.double().square().sum()) for t in many)
    assert abs(float(ops.squared_norm(many)) - want) <= 64 * U * want
    mixed_types = [many[0], many[1].bfloat16(), many[2].half(), many[3]]
    want = sum(float(t.double().square().sum()) for t in mixed_types)
    assert abs(float(ops.squared_norm(mixed_types)) - want) <= 64 * U * want
    strided = [big[:400].view(20, 20).t(), big[:400].view(20, 20)[:, 3:9], big[0].expand(7)]
    want = sum(float(t.double().square().sum()) for t in strided)
    assert abs(float(ops.squared_norm(strided)) - want) <= 64 * U * want
    assert float(ops.squared_norm([big[:0]])) == 0.0
    assert math.isnan(float(ops.squared_norm([torch.tensor([1.0, float("nan")], device="cuda")])))
    assert math.isinf(float(ops.squared_norm([torch.tensor([1.0, float("inf")], device="cuda")])))


# ---- dequantize -------------------------------------------------------------------------------------
@pytest.mark.parametrize("n", [0, 1, 31, 32, 33, 1000, 70001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_dequantize(ops, n, dtype):
    gen = torch.Generator(device="cuda").manual_seed(12)
    codes = torch.randint(0, 256, (n,), generator=gen, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn)
    low, high = (10, 247) if dtype != torch.float16 else (115, 134)  # 448 times the next one is no fp32 number
    scales = torch.randint(low, high, (-(-n // 32),), generator=gen, device="cuda", dtype=torch.uint8).view(torch.float8_e8m0fnu)
    got = ops.dequantize_blocks(codes, scales, dtype)
    want = codes.double() * scales.double().repeat_interleave(32)[:n]
    assert got.dtype == dtype and torch.equal(got.isnan(), want.isnan())
    fine = ~want.isnan()
    assert torch.equal(got[fine].double(), want[fine].float().to(dtype).double())
    if dtype != torch.float16 and n:
        assert torch.equal(got[fine].double(), want[fine])  # exact


# ---- the optimizer ----------------------------------------------------------------------------------
def model(dtype=torch.float32):
    torch.manual_seed(0)
    return torch.nn.Sequential(torch.nn.Linear(40, 70), torch.nn.LayerNorm(70), torch.nn.Tanh(), torch.nn.Linear(70, 3)).cuda().to(dtype)


def train(net, opt, steps, max_norm=None, seed=1):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    losses = []
    for _ in range(steps):
        x = torch.randn(64, 40, generator=gen, device="cuda").to(next(net.parameters()).dtype)
        target = torch.stack([x[:, 0] * x[:, 1], x[:, 2].abs(), x[:, 3:6].sum(1)], 1)
        loss = (net(x) - target).square().mean()
        opt.zero_grad()
        loss.backward()
        if max_norm is not None:
            torch.nn.utils.clip_grad_norm_(net.parameters(), max_norm)
        opt.step()
        losses.append(float(loss.detach()))
    return losses


@pytest.mark.parametrize("max_norm", [None, 0.2])
def test_optimizer_follows_torch(ops, max_norm):
    a, b = model(), model()
    groups = lambda net: [{"params": [p for p in net.parameters() if p.dim() > 1], "weight_decay": 0.1},  # noqa: E731
                          {"params": [p for p in net.parameters() if p.dim() < 2], "weight_decay": 0.0, "lr": 2e-3}]
    ours = ops.AdamW(groups(a), lr=1e-3, max_norm=max_norm)
    theirs = torch.optim.AdamW(groups(b), lr=1e-3)
    x = train(a, ours, 40)
    y = train(b, theirs, 40, max_norm)
    assert max(abs(u - v) for u, v in zip(x, y)) < 1e-3
    for p, q in zip(a.parameters(), b.parameters()):
        assert float((p - q).abs().max()) < 2e-3  # 40 steps of 1e-3, whose signs may differ where a gradient is noise
        assert float((p - q).square().mean().sqrt()) < 1e-4


def test_optimizer_in_8_bits_learns_like_32(ops):
    results = []
    for bits, dtype in ((32, torch.float32), (8, torch.float32), (8, torch.bfloat16)):
        net = model(dtype)
        results.append(sum(train(net, ops.AdamW(net.parameters(), lr=3e-3, state_bits=bits), 400)[-50:]) / 50)
    assert results[0] < 0.45 and results[1] < 1.1 * results[0] + 0.02 and results[2] < 1.2 * results[0] + 0.05, results


@pytest.mark.parametrize("bits", [32, 8])
def test_optimizer_state_dict(ops, bits):
    a = model()
    opt = ops.AdamW(a.parameters(), lr=1e-3, state_bits=bits, seed=5)
    train(a, opt, 5)
    b = copy.deepcopy(a)
    again = ops.AdamW(b.parameters(), lr=7.0, state_bits=bits, seed=5)
    again.load_state_dict(copy.deepcopy(opt.state_dict()))
    assert train(a, opt, 5, seed=2) == train(b, again, 5, seed=2)
    assert all(torch.equal(p, q) for p, q in zip(a.parameters(), b.parameters()))
    twin = copy.deepcopy(opt)
    assert twin.state_bits == bits and twin.seed == 5
    other = ops.AdamW(b.parameters(), state_bits=40 - bits)
    with pytest.raises(ValueError, match="another optimizer"):
        other.load_state_dict(opt.state_dict())


def test_optimizer_sees_only_what_has_a_gradient(ops):
    a, b = torch.nn.Parameter(torch.ones(10, device="cuda")), torch.nn.Parameter(torch.ones(10, device="cuda"))
    empty = torch.nn.Parameter(torch.ones(0, device="cuda"))
    opt = ops.AdamW([a, b, empty], lr=0.1)
    opt.step()
    a.grad, empty.grad = torch.ones(10, device="cuda"), torch.ones(0, device="cuda")
    version = a._version
    opt.step()
    assert bool((b == 1).all()) and not opt.state[b] and bool((a != 1).all()) and a._version > version
    b.grad = torch.ones(10, device="cuda")
    opt.step()  # b begins at step 1 beside a's step 2
    assert opt.state[a]["step"] == 2 and opt.state[b]["step"] == 1
    # laid out otherwise
    c = torch.nn.Parameter(torch.randn(6, 8, device="cuda").t())
    c.grad = torch.randn(6, 8, device="cuda").t().contiguous()
    want = formula(c.detach(), c.grad, torch.zeros_like(c), torch.zeros_like(c), 1, 0.1, (0.9, 0.999), 1e-8, 0.01)
    ops.AdamW([c], lr=0.1).step()
    close(c.detach(), want[0], want[3], "transposed")
    # a closure
    opt = ops.AdamW([a], lr=0.1)
    assert opt.step(lambda: 5) == 5


def test_steps_on_another_stream(ops):
    gen = torch.Generator(device="cuda").manual_seed(13)
    p, g = make([50_000], torch.float32, 1, gen)[0], make([50_000], torch.float32, 1, gen)[0]
    results = []
    for stream in (torch.cuda.current_stream(), torch.cuda.Stream()):
        q, states = p.clone(), new_states(ops, 50_000)
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            call(ops, [q], [g], [states], 1, squared_norm=ops.squared_norm([g]), max_norm=1.0)
        torch.cuda.synchronize()
        results.append(q)
    assert torch.equal(*results)


def test_steps_in_a_graph(ops):
    gen = torch.Generator(device="cuda").manual_seed(14)
    start, g = make([3000, 77], torch.float32, 1, gen), make([3000, 77], torch.float32, 1, gen)

    def step(ps, states):
        call(ops, ps, g, states, 3, squared_norm=ops.squared_norm(g), max_norm=1.0)

    ps, states = [p.clone() for p in start], [new_states(ops, n) for n in (3000, 77)]
    step(ps, states)
    eager = []
    for _ in range(3):
        step(ps, states)
        eager.append([p.clone() for p in ps])
    ps, states = [p.clone() for p in start], [new_states(ops, n) for n in (3000, 77)]
    step(ps, states)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(ps, states)
    for want in eager:
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(ps, want))
        float(ops.squared_norm(g))  # the program's own work between the replays
    opt = ops.AdamW([torch.nn.Parameter(start[0].clone())])
    opt.param_groups[0]["params"][0].grad = g[0]
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(graph):
            opt.step()


def test_refusals(ops):
    p, g, m, v = (torch.ones(64, device="cuda") for _ in range(4))
    codes, scales = new_states(ops, 64)[:2]
    roots, root_scales = new_states(ops, 64)[:2]

    def step(p=p, g=g, m=m, v=v, **more):
        ops.adamw_step([p], [g], [m], [v], **{**dict(step=1, lr=1e-3), **more})

    def step8(p=p, g=g, m=codes, ms=scales, v=roots, vs=root_scales, **more):
        ops.adamw_step_8bit([p], [g], [m], [ms], [v], [vs], **{**dict(step=1, lr=1e-3, seed=1), **more})

    for wrong, error in [
        (dict(p=p.half()), "params"), (dict(p=p.double()), "params"), (dict(p=p.cpu()), "GPU"), (dict(g=g.double()), "grads"), (dict(g=g.cpu()), "GPU"),
        (dict(g=g[:63]), "laid out"), (dict(m=m.half()), "exp_avgs"), (dict(v=v[:63]), "laid out"), (dict(step=0), "first step"),
        (dict(betas=(1.0, 0.9)), "betas"), (dict(lr=-1.0), "lr"), (dict(eps=float("inf")), "finite"), (dict(grad_scale=-1.0), "grad_scale"),
        (dict(squared_norm=torch.ones((), device="cuda")), "together"), (dict(max_norm=1.0), "together"),
        (dict(squared_norm=torch.ones(2, device="cuda"), max_norm=1.0), "squared_norm"), (dict(copies=[]), "copies"),
        (dict(copies=[torch.ones(64, device="cuda")]), "copies"), (dict(p=p.bfloat16(), copies=[p.bfloat16()]), "copies"),
        (dict(p=torch.ones(64, 2, device="cuda")[:, 0]), "dense"),
    ]:
        with pytest.raises((TypeError, ValueError, RuntimeError), match=error):
            step(**wrong)
    for wrong, error in [(dict(m=m), "exp_avgs"), (dict(ms=scales[:1]), "exp_avg_scales"), (dict(v=v), "exp_avg_roots"),
                         (dict(vs=root_scales.view(torch.uint8)), "scales"), (dict(seed=None), "seed"), (dict(m=codes[:60]), "exp_avgs")]:
        with pytest.raises((TypeError, ValueError), match=error):
            step8(**wrong)
    with pytest.raises(ValueError, match="overlap"):
        ops.adamw_step([p, p[32:]], [g, g[32:]], [m, m[32:]], [v, v[32:]], step=1, lr=1e-3)
    with pytest.raises(TypeError, match="one dtype"):
        ops.adamw_step([p, p.bfloat16()], [g, g], [m, m], [v, v], step=1, lr=1e-3)
    with pytest.raises(ValueError, match="tensors for"):
        ops.adamw_step([p], [], [m], [v], step=1, lr=1e-3)
    ops.adamw_step([], [], [], [], step=1, lr=1e-3)
    assert bool((p == 1).all()) and bool((m == 1).all()), "a refused call wrote something"
    with pytest.raises(ValueError):
        ops.squared_norm([])
    with pytest.raises(TypeError):
        ops.squared_norm([p.double()])
    with pytest.raises(TypeError):
        ops.dequantize_blocks(p, scales)
    with pytest.raises(ValueError):
        ops.dequantize_blocks(codes, scales[:1])
    for wrong in (dict(lr=-1.0), dict(betas=(0.9, 1.0)), dict(state_bits=16), dict(max_norm=-1.0)):
        with pytest.raises(ValueError):
            ops.AdamW([torch.nn.Parameter(p.clone())], **wrong)
