"""The operators of ``odc_amd.ops`` as cases to be measured: layer norm forward and backward, the AdamW step
over many tensors with states in 32 bits or 8, and the squared norm of many tensors.

``run`` is one pass: where ``own`` is false in elementary torch operations in 32 bits, where it is true through
the package's public entry points. The tensors of a list are views of one flat buffer, as the shards in a
symmetric arena are, so the plain form too goes over all of them at once.

The formulas. Layer norm of a row of N: ``y = (x - mean) * rstd * w + b``, ``rstd = 1 / sqrt(var + eps)``. With a
residual: ``total = x + residual`` in the tensors' type, which is handed on, and ``y`` is the norm of it. AdamW:
``g = grad * min(1, max_norm / (sqrt(squared norm) + 1e-6))``, ``m = b1 m + (1 - b1) g``, ``v = b2 v + (1 - b2) g^2``,
``p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)``.

States in 8 bits: m and the root of v as e4m3 values (3 bits of mantissa, at most 448) in blocks of 32 with a
power of two as scale, the smallest that keeps the block's largest value within 448. A value between two of these is
stored as one of them by a given random number: m so that its expectation is m, the root so that the expectation of
its square is v; a v that is not zero is not stored as zero. The random number of element i of tensor k in the step
with seed s is ``word = mix(i + mix(s + k * 0x9E3779B1))``, its low half for m, its high half for the root, and for a
parameter in bf16 the low half of ``mix(word ^ 0x5BF03635)``, added below the 16 bits that stay. A half h chooses
the upper code where ``(h + 0.5) / 65536`` is less than the share of the way.
"""

import itertools
import math
import random

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
EPS_NORM = 1e-5
LR, BETA1, BETA2, EPS, DECAY, MAX_NORM = 3e-4, 0.9, 0.999, 1e-8, 0.1, 1.0
FIRST_STEP = 100
BLOCK = 32  # elements of a state in 8 bits that share a scale
LOWEST_SCALE = 10  # a scale is at least 2^(10 - 127): its smallest multiple is no subnormal number


# ---- cases --------------------------------------------------------------------------------------
def _norm_case(rows, n, dtype, wdtype, add, train, pad=0):
    return {"op": "layer_norm", "rows": rows, "n": n, "dtype": dtype, "wdtype": wdtype, "add": add, "train": train, "pad": pad}


def _sizes(kind, count=0, low=0, high=0, sizes_seed=0, align=256):
    return {"sizes": kind, "count": count, "low": low, "high": high, "sizes_seed": sizes_seed, "align": align}


def _adamw_case(bits, param, grad, copy, clip, **sizes):
    return {"op": "adamw", "bits": bits, "param": param, "grad": grad, "copy": copy, "clip": clip, **sizes}


def listed():
    return [
        # The toy transformer's norm (width 256, 32 sequences of 64) without gradients, as an evaluation pass calls
        # it: a megabyte, all latency.
        dict(_norm_case(2048, 256, "fp32", "fp32", False, False), name="norm_toy_forward"),
        # One microbatch (2 x 2048 tokens) through a norm of the 4096 wide decoder layer in training: everything in
        # bf16, as FSDP's mixed precision hands the parameters out.
        dict(_norm_case(4096, 4096, "bf16", "bf16", False, True), name="norm_4096_train"),
        # The same behind a residual addition, the weights left in fp32.
        dict(_norm_case(4096, 4096, "bf16", "fp32", True, True), name="add_norm_4096_train"),
        # Odd width in fp16, rows that are slices of a wider tensor and start at no boundary.
        dict(_norm_case(1000, 1001, "fp16", "fp32", False, True, pad=37), name="norm_odd_slice_train"),
        # The largest: 16384 tokens of the layer's wide side (14336), with the residual addition.
        dict(_norm_case(16384, 14336, "bf16", "bf16", True, True), name="add_norm_14336_train"),
        # The toy transformer's 25 parameters, sharded over 8 ranks, full precision: launches are all of it.
        dict(_adamw_case(32, "fp32", "fp32", "", False, **_sizes("toy")), name="adamw_toy"),
        # A rank's shards of the decoder layer (W = 8) as FSDP2 keeps them: fp32 shards and gradients, clipping,
        # and the bf16 copy that the next minibatch's gathers read.
        dict(_adamw_case(32, "fp32", "fp32", "bf16", True, **_sizes("layer")), name="adamw_layer_clip_copy"),
        # A rank's shards of the whole 8.03 G parameter model (W = 8), one flat parameter for each of its 34 units.
        dict(_adamw_case(32, "fp32", "fp32", "", False, **_sizes("model")), name="adamw_model"),
        # The layer's shards with states in 8 bits.
        dict(_adamw_case(8, "fp32", "fp32", "", True, **_sizes("layer")), name="adamw8_layer_clip"),
        # Forty uneven flat parameters, everything in bf16 and the states in 8 bits.
        dict(_adamw_case(8, "bf16", "bf16", "", False, **_sizes("list", 40, 341, 4_893_355, 7)), name="adamw8_uneven_bf16"),
        # The norm of 300 small gradients (biases, norms, adapters), packed without gaps.
        dict({"op": "squared_norm", "grad": "fp32", **_sizes("list", 300, 64, 65_536, 3, align=1)}, name="squared_norm_many_small"),
        # The norm of the whole model's gradients on one rank, in bf16.
        dict({"op": "squared_norm", "grad": "bf16", **_sizes("model")}, name="squared_norm_model"),
    ]


def _log_uniform(rng, low, high):
    return int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))


def draw(rng):
    op = rng.choice(["layer_norm", "layer_norm", "adamw", "adamw", "squared_norm"])
    if op == "layer_norm":
        n = _log_uniform(rng, 32, 20_000)
        rows = _log_uniform(rng, 1, min(32_768, 16384 * 14336 // n))
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        return _norm_case(rows, n, dtype, rng.choice([dtype, "fp32"]), rng.random() < 0.4, rng.random() < 0.7,
                          rng.choice([0, 0, 0, _log_uniform(rng, 1, 200)]))
    count = _log_uniform(rng, 1, 400)
    high = _log_uniform(rng, 1000, max(2000, 150_000_000 // count))
    # states in 8 bits have blocks that begin with each tensor; the others may lie packed
    sizes = _sizes("list", count, max(1, high // rng.choice([1, 4, 64, 1000])), high, rng.randrange(1 << 20))
    if op == "squared_norm":
        return {"op": op, "grad": rng.choice(["fp32", "bf16", "fp16"]), **dict(sizes, align=rng.choice([1, 256]))}
    bits = rng.choice([32, 8])
    param = rng.choice(["fp32", "fp32", "bf16"])
    if bits == 32:
        sizes["align"] = rng.choice([1, 256])
    return _adamw_case(bits, param, rng.choice(["fp32", "bf16", "fp16"]) if param == "fp32" else "bf16",
                       rng.choice(["", "bf16", "fp16"]) if param == "fp32" else "", rng.random() < 0.5, **sizes)


def _numels(case):
    """The elements of every tensor of a list."""
    if case["sizes"] == "toy":
        block = [(256,), (256,), (768, 256), (256, 256), (256,), (256,), (1024, 256), (1024,), (256, 1024), (256,)]
        shapes = [(1024, 256), (64, 256), *block, *block, (256,), (256,), (1024, 256)]
        return [math.prod(s) // 8 for s in shapes]
    if case["sizes"] == "layer":
        h, f, kv = 4096, 14336, 1024
        return [n // 8 for n in (h, h * h, kv * h, kv * h, h * h, h, f * h, f * h, h * f)]
    if case["sizes"] == "model":
        h, layer, vocab = 4096, 218_112_000, 128256
        return [n // 8 for n in (vocab * h, *[layer] * 32, h + vocab * h)]
    rng = random.Random(case["sizes_seed"])
    return [_log_uniform(rng, case["low"], case["high"]) for _ in range(case["count"])]


def work(case):
    """Every input read once, every output written once."""
    if case["op"] == "layer_norm":
        e, ws, big = DTYPES[case["dtype"]].itemsize, DTYPES[case["wdtype"]].itemsize, case["rows"] * case["n"]
        streams = 4 if case["add"] else 2  # x, y; residual, total
        if case["train"]:
            streams += 3 if case["add"] else 2  # dy, dx; dtotal
        return {"bytes": streams * big * e + (4 if case["train"] else 2) * case["n"] * ws, "flops": big * (22 if case["train"] else 8)}
    n = sum(_numels(case))
    if case["op"] == "squared_norm":
        return {"bytes": n * DTYPES[case["grad"]].itemsize + 4, "flops": 2 * n}
    per = 2 * DTYPES[case["param"]].itemsize + DTYPES[case["grad"]].itemsize + (DTYPES[case["copy"]].itemsize if case["copy"] else 0)
    # states read and written; those in 8 bits are also read once more as bf16 values (the outputs of run)
    per += 16 if case["bits"] == 32 else 4 * (1 + 1 / BLOCK) + 2 * (1 + 1 / BLOCK + 2)
    return {"bytes": n * per, "flops": n * (16 if case["bits"] == 32 else 40)}


# ---- preparation --------------------------------------------------------------------------------
def _starts(numels, align):
    """Where the tensors of a list begin in their flat buffer, at multiples of ``align`` elements, and where it ends."""
    return [0, *itertools.accumulate(-(-n // align) * align for n in numels)]


def _scales(x):
    """The biased exponent k of every block's scale: the smallest with largest / 2^(k - 127) <= 448 = 1.75 * 2^8."""
    largest = x.view(-1, BLOCK).abs().amax(1)
    return ((largest.view(torch.int32) + 0x1FFFFF >> 23) - 8).clamp(min=LOWEST_SCALE)


def _scaled(x, k):
    return (x.view(-1, BLOCK) * (254 - k << 23).view(torch.float32)[:, None]).view(-1)


def _nearest_codes(x):
    """x as e4m3 values and the scales of its blocks: states such as earlier steps leave."""
    k = _scales(x)
    return _scaled(x, k).to(torch.float8_e4m3fn), k.to(torch.uint8).view(torch.float8_e8m0fnu)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    s = {"case": case}
    if case["op"] == "layer_norm":
        rows, n, dtype, wdtype = case["rows"], case["n"], DTYPES[case["dtype"]], DTYPES[case["wdtype"]]

        def activations(scale, grad):
            # a residual stream has a mean of its own and channels that stand out
            wide = (randn(rows, n + case["pad"]) * randn(n + case["pad"]).mul_(0.5).exp_() * scale + 0.3).to(dtype)
            t = wide[:, case["pad"] // 2 : case["pad"] // 2 + n]
            return t.requires_grad_(grad and case["train"])

        s["x"] = activations(1.5, True)
        if case["add"]:
            s["residual"] = activations(2.0, True)
        if case["train"]:
            s["dy"] = (randn(rows, n) * 1e-2).to(dtype)
            if case["add"]:
                s["dtotal"] = (randn(rows, n) * 1e-2).to(dtype)
        s["w"] = (1 + 0.2 * randn(n)).to(wdtype).requires_grad_(case["train"])
        s["b"] = (0.1 * randn(n)).to(wdtype).requires_grad_(case["train"])
        return s

    numels = s["numels"] = _numels(case)

    def views(flat, unit=1):
        return [flat[a // unit : a // unit + -(-n // unit)] for a, n in zip(s["starts"], numels)]

    def values(dtype, scale):
        flat = torch.zeros(total, dtype=dtype, device="cuda")
        for view in views(flat):
            # gradients of different tensors differ in size
            view.copy_(randn(view.numel()).mul_(scale * math.exp((len(numels) + view.numel()) % 5 - 2)))
        return flat

    *s["starts"], total = _starts(numels, case["align"])
    s["grad_flat"] = values(DTYPES[case["grad"]], 1e-3)
    s["grads"] = views(s["grad_flat"])
    if case["op"] == "squared_norm":
        return s
    s["step"] = FIRST_STEP
    s["param_flat"] = values(DTYPES[case["param"]], 0.02)
    s["params"] = views(s["param_flat"])
    s["copy_flat"] = torch.zeros_like(s["param_flat"], dtype=DTYPES[case["copy"]]) if case["copy"] else None
    s["copies"] = views(s["copy_flat"]) if case["copy"] else None
    m, root = values(torch.float32, 3e-4), values(torch.float32, 8e-4).abs_()
    if case["bits"] == 32:
        s["m_flat"], s["v_flat"] = m, root.square_()
        s["ms"], s["vs"] = views(m), views(s["v_flat"])
        return s
    # the plan of the flat buffer: how far the places of each tensor reach
    edges = torch.tensor([*s["starts"], total], device="cuda")
    s["lengths"], s["edges"] = edges[1:] - edges[:-1], edges[:-1]
    s["m_flat"], s["m_scale_flat"] = _nearest_codes(m)
    s["root_flat"], s["root_scale_flat"] = _nearest_codes(root)
    s["ms"], s["roots"] = views(s["m_flat"]), views(s["root_flat"])
    s["m_scales"], s["root_scales"] = views(s["m_scale_flat"], BLOCK), views(s["root_scale_flat"], BLOCK)
    return s


# ---- one pass -----------------------------------------------------------------------------------
def run(s):
    op = s["case"]["op"]
    if own:
        from odc_amd import ops

        if op == "layer_norm":
            return _own_layer_norm(ops, s)
        if op == "squared_norm":
            return {"squared_norm": ops.squared_norm(s["grads"])}
        return _own_adamw(ops, s)
    with torch.no_grad():
        if op == "layer_norm":
            return _plain_layer_norm(s)
        if op == "squared_norm":
            return {"squared_norm": s["grad_flat"].float().square().sum()}
        return _plain_adamw(s)


def _own_layer_norm(ops, s):
    case, shape = s["case"], (s["case"]["n"],)
    if case["add"]:
        y, total = ops.add_layer_norm(s["x"], s["residual"], shape, s["w"], s["b"], EPS_NORM)
        if not case["train"]:
            return {"y": y, "total": total}
        dx, dw, db = torch.autograd.grad((y, total), (s["x"], s["w"], s["b"]), (s["dy"], s["dtotal"]))
        return {"y": y, "total": total, "dx": dx, "dw": dw, "db": db}
    y = ops.layer_norm(s["x"], shape, s["w"], s["b"], EPS_NORM)
    if not case["train"]:
        return {"y": y}
    dx, dw, db = torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["dy"])
    return {"y": y, "dx": dx, "dw": dw, "db": db}


def _plain_layer_norm(s):
    case, dtype, wdtype = s["case"], s["x"].dtype, s["w"].dtype
    out = {}
    if case["add"]:
        out["total"] = (s["x"].float() + s["residual"].float()).to(dtype)
        x = out["total"].float()
    else:
        x = s["x"].float()
    w = s["w"].float()
    centred = x - x.mean(1, keepdim=True)
    rstd = (centred.square().mean(1, keepdim=True) + EPS_NORM).rsqrt()
    xhat = centred * rstd
    out["y"] = (xhat * w + s["b"].float()).to(dtype)
    if not case["train"]:
        return out
    dy = s["dy"].float()
    out["dw"], out["db"] = (dy * xhat).sum(0).to(wdtype), dy.sum(0).to(wdtype)
    h = dy * w
    dx = (h - h.mean(1, keepdim=True) - xhat * (h * xhat).mean(1, keepdim=True)) * rstd
    if case["add"]:
        dx += s["dtotal"].float()
    out["dx"] = dx.to(dtype)
    return out


def _own_adamw(ops, s):
    case = s["case"]
    s["step"] += 1
    sq = ops.squared_norm(s["grads"]) if case["clip"] else None
    numbers = dict(step=s["step"], lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY, squared_norm=sq,
                   max_norm=MAX_NORM if case["clip"] else None, copies=s["copies"])
    out = {"param": s["param_flat"]}
    if case["clip"]:
        out["squared_norm"] = sq
    if case["copy"]:
        out["copy"] = s["copy_flat"]
    if case["bits"] == 32:
        ops.adamw_step(s["params"], s["grads"], s["ms"], s["vs"], **numbers)
        return {**out, "m": s["m_flat"], "v": s["v_flat"]}
    ops.adamw_step_8bit(s["params"], s["grads"], s["ms"], s["m_scales"], s["roots"], s["root_scales"], seed=s["step"], **numbers)
    return {**out, "m": ops.dequantize_blocks(s["m_flat"], s["m_scale_flat"], torch.bfloat16),
            "root": ops.dequantize_blocks(s["root_flat"], s["root_scale_flat"], torch.bfloat16)}


def _plain_adamw(s):
    case = s["case"]
    s["step"] += 1
    t, out = s["step"], {"param": s["param_flat"]}
    g = s["grad_flat"].float()
    if case["clip"]:
        out["squared_norm"] = g.square().sum()
        g = g * (MAX_NORM / (out["squared_norm"].sqrt() + 1e-6)).clamp(max=1)
    if case["bits"] == 32:
        m = s["m_flat"].mul_(BETA1).add_(g * (1 - BETA1))
        v = s["v_flat"].mul_(BETA2).add_(g.square() * (1 - BETA2))
        root = v.sqrt()
        out |= {"m": m, "v": v}
    else:
        m = _read_codes(s["m_flat"], s["m_scale_flat"]).mul_(BETA1).add_(g * (1 - BETA1))
        v = _read_codes(s["root_flat"], s["root_scale_flat"]).square_().mul_(BETA2).add_(g.square() * (1 - BETA2))
        root = v.sqrt()
    update = m / (root / math.sqrt(1 - BETA2**t) + EPS)
    p = s["param_flat"].float() * (1 - LR * DECAY) - update * (LR / (1 - BETA1**t))
    if case["bits"] == 8:
        keys = _mix(torch.arange(len(s["numels"]), device="cuda") * 0x9E3779B1 + t & 0xFFFFFFFF)
        spread = torch.repeat_interleave(keys - s["edges"], s["lengths"], output_size=g.numel())
        words = _mix(spread + torch.arange(g.numel(), device="cuda") & 0xFFFFFFFF)
        _write_codes(m, words & 0xFFFF, s["m_flat"], s["m_scale_flat"], squares=False)
        _write_codes(root, words >> 16, s["root_flat"], s["root_scale_flat"], squares=True)
        out["m"] = _read_codes(s["m_flat"], s["m_scale_flat"]).bfloat16()
        out["root"] = _read_codes(s["root_flat"], s["root_scale_flat"]).bfloat16()
        if p.dtype != s["param_flat"].dtype:
            p = ((p.view(torch.int32) + (_mix(words ^ 0x5BF03635) & 0xFFFF).int()) & ~0xFFFF).view(torch.float32)
    s["param_flat"].copy_(p)
    if case["copy"]:
        out["copy"] = s["copy_flat"].copy_(p)
    return out


def _mix(x):
    """A number of 32 bits from each of x, as 64 bit integers: every bit of it depends on all of x's."""
    x = ((x ^ (x >> 16)) * 0xB7E15163) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0x9E3779B1) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _read_codes(codes, scales):
    return (codes.float().view(-1, BLOCK) * scales.float()[:, None]).view(-1)


def _write_codes(x, chance, codes, scales, squares):
    """Stores x, each value by its 16 random bits as one of the two codes beside it."""
    k = _scales(x)
    size = _scaled(x.abs(), k)
    if squares:
        size = torch.where(size > 0, size.clamp(min=2.0**-9), size)
    step = (size.clamp(min=2.0**-6).view(torch.int32) & 0x7F800000).view(torch.float32) / 8  # 3 bits of mantissa stay
    below = (size / step).floor() * step
    share, whole = size - below, step
    if squares:
        share, whole = share * (size + below), step * (below + below + step)
    size = below + torch.where((chance.float() + 0.5) * whole < share * 65536, step, 0)
    codes.copy_(torch.copysign(size, x))
    scales.view(torch.uint8).copy_(k)


# ---- the definition in 64 bits ------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "layer_norm":
        with torch.no_grad():
            x, w = s["x"].double(), s["w"].double()
            out = {}
            if case["add"]:
                x = (x + s["residual"].double()).to(s["x"].dtype).double()  # the sum is defined in the tensors' type
                out["total"] = x
            mean = x.sum(1) / case["n"]
            var = ((x - mean[:, None]) ** 2).sum(1) / case["n"]
            sigma = torch.sqrt(var + EPS_NORM)[:, None]
            z = (x - mean[:, None]) / sigma
            out["y"] = z * w + s["b"].double()
            if case["train"]:
                dy = s["dy"].double()
                out["dw"], out["db"] = torch.sum(z * dy, 0), torch.sum(dy, 0)
                # the Jacobian of z: (identity - ones/N - z z^T / N) / sigma
                a = dy * w
                out["dx"] = (a - a.sum(1, True) / case["n"] - z * ((a * z).sum(1, True) / case["n"])) / sigma
                if case["add"]:
                    out["dx"] += s["dtotal"].double()
            return out
    sq = torch.zeros((), dtype=torch.float64, device="cuda")
    for g in s["grads"]:
        sq += (g.double() ** 2).sum()
    if case["op"] == "squared_norm":
        return {"squared_norm": sq}
    t, n = FIRST_STEP + 1, s["param_flat"].numel()
    names = ["param", "m", "v" if case["bits"] == 32 else "root"] + (["copy"] if case["copy"] else [])
    out = {name: torch.zeros(n, dtype=torch.float64, device="cuda") for name in names}
    factor = min(1.0, MAX_NORM / (math.sqrt(float(sq)) + 1e-6)) if case["clip"] else 1.0

    def mixed(x):
        for shift, odd in ((16, 0xB7E15163), (15, 0x9E3779B1)):
            x = (x ^ (x >> shift)) * odd & 0xFFFFFFFF
        return x ^ (x >> 16)

    def value(codes, scales):
        return codes.double() * torch.repeat_interleave(scales.double(), BLOCK)[: codes.numel()]

    def stored(x, chance, power):
        """x as its codes stand for it; chance in [0, 1)."""
        blocks = torch.nn.functional.pad(x.abs(), (0, -x.numel() % BLOCK)).view(-1, BLOCK)
        top = blocks.amax(1).clamp(min=1e-300)
        scale = torch.exp2(torch.ceil(torch.log2(top / 448)).clamp(min=LOWEST_SCALE - 127))
        scale = torch.repeat_interleave(scale, BLOCK)[: x.numel()]
        a = x.abs() / scale
        if power == 2:
            a = torch.where(a > 0, a.clamp(min=2.0**-9), a)
        ulp = torch.exp2(torch.floor(torch.log2(a.clamp(min=2.0**-6))) - 3)
        low = torch.floor(a / ulp) * ulp
        p = (a**power - low**power) / ((low + ulp) ** power - low**power)
        return torch.sign(x) * scale * torch.where(chance < p, low + ulp, low)

    for k, at in enumerate(s["starts"]):
        p, g = s["params"][k].double(), s["grads"][k].double() * factor
        if case["bits"] == 32:
            m, v = s["ms"][k].double(), s["vs"][k].double()
        else:
            m, v = value(s["ms"][k], s["m_scales"][k]), value(s["roots"][k], s["root_scales"][k]) ** 2
        m = BETA1 * m + (1 - BETA1) * g
        v = BETA2 * v + (1 - BETA2) * g * g
        p = p - LR * DECAY * p - LR * (m / (1 - BETA1**t)) / (torch.sqrt(v / (1 - BETA2**t)) + EPS)
        here = slice(at, at + p.numel())
        if case["bits"] == 32:
            out["v"][here] = v
        else:
            word = mixed(torch.arange(p.numel(), device="cuda") + mixed(t + k * 0x9E3779B1 & 0xFFFFFFFF) & 0xFFFFFFFF)
            m, out["root"][here] = stored(m, (word % 65536 + 0.5) / 65536, 1), stored(torch.sqrt(v), (word // 65536 + 0.5) / 65536, 2)
            if case["param"] == "bf16":
                ulp = torch.exp2(torch.floor(torch.log2(p.abs().clamp(min=2.0**-126))) - 7)
                p = torch.sign(p) * ulp * torch.floor(p.abs() / ulp + (mixed(word ^ 0x5BF03635) % 65536) / 65536)
        out["param"][here], out["m"][here] = p, m
        if case["copy"]:
            out["copy"][here] = p
    if case["clip"]:
        out["squared_norm"] = sq
    return out
