"""Low-bit products and the optimiser's step as measurable cases: what trains a layer's weights and what serves them in
4 bits, beside the dense operators of ``perf/operators.py``.

Both keep numbers in blocks of 32 with a power of two as the block's scale (one byte, exponent + 127): elements of 4 bits
(sign, 2 bits of exponent, 1 of fraction: 0, 0.5, 1, 1.5, 2, 3, 4, 6) for products, of 8 bits (sign, 4, 3) for an
optimiser's states.

A case is a plain dict:

    op      "quant"        rows into 4-bit codes and block scales, and back into the values that those stand for
            "matmul"       4-bit codes times 4-bit weights, with the scales of both sides' blocks
            "norm_matmul"  serving: residual's addition, root-mean-square norm into 4-bit codes, product with 4-bit weights
            "adamw"        one AdamW step over a list of tensors; states in 32 bits or in 8
    rows, width            rows and features; `x`: their type, `out`: the values' type                   (quant)
    m, n, k                rows, output channels, inner length; `out`; `bias`                            (matmul)
    m, n, k, x, res, out   rows, output channels, features; types of the input and the residual          (norm_matmul)
    elements, tensors      elements in all, tensors that share them out                                  (adamw)
    p, g, copy             types of the parameters, their gradients and the copies for the next forward pass ("none": no copies)
    bits, step, clip       of the states; the step's number; whether a factor on the gradients comes from the GPU

Where `own` is false, `run` computes the same in elementary torch operations in 32 bits.
"""
import math
import os
import random
import sys

import torch

#: Set by who measures: true for the library's kernels, false for the plain form.
own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2, "none": 0}
EPS = 1e-5
BLOCK = 32

LR, BETAS, ADAM_EPS, DECAY, SEED = 1e-3, (0.9, 0.999), 1e-8, 0.01, 20

#: What the largest listed cases cost: no drawn case has more of either.
MOST_BYTES = 28 << 27
MOST_FLOPS = 2 * 8192 ** 3


def listed():
    return [
        # the activations of a few tokens: latency
        {"name": "quant 64 x 4096", "op": "quant", "rows": 64, "width": 4096, "x": "f16", "out": "f16"},
        # what an aggregation hands on, of a width off the blocks
        {"name": "quant 250k x 300", "op": "quant", "rows": 250_001, "width": 300, "x": "f32", "out": "bf16"},
        # a large weight's forward values in training that knows of its 4 bits
        {"name": "quant 16k x 4096", "op": "quant", "rows": 16384, "width": 4096, "x": "bf16", "out": "bf16"},
        # serving, one token: bound by the weights
        {"name": "matmul 1 x 4096 x 4096", "op": "matmul", "m": 1, "n": 4096, "k": 4096, "out": "f16", "bias": False},
        # a ragged batch: rows and channels off the tiles, k off the blocks
        {"name": "matmul 500 x 1000 x 2010", "op": "matmul", "m": 500, "n": 1000, "k": 2010, "out": "f32", "bias": True},
        # a large batch through a wide layer: bound by arithmetic
        {"name": "matmul 8k x 8k x 8k", "op": "matmul", "m": 8192, "n": 8192, "k": 8192, "out": "bf16", "bias": False},
        # serving, one token through a whole projection
        {"name": "norm_matmul 1 x 4096 x 4096", "op": "norm_matmul", "m": 1, "n": 4096, "k": 4096, "x": "f16", "res": "f16",
         "out": "f16"},
        # a graph layer's projection over all nodes: float32 sums of the aggregation, residual in 16 bits
        {"name": "norm_matmul 1m x 256 x 128", "op": "norm_matmul", "m": 1 << 20, "n": 256, "k": 128, "x": "f32", "res": "f16",
         "out": "f16"},
        # a small layer's table, norm and projection: latency
        {"name": "adamw 3 of 34k", "op": "adamw", "elements": 33_856, "tensors": 3, "p": "f32", "g": "f32", "copy": "none",
         "bits": 32, "step": 1, "clip": False},
        # the many tensors of a deep model, gradients and copies in 16 bits, clipped
        {"name": "adamw 8 bits 148 of 85m", "op": "adamw", "elements": 85_000_001, "tensors": 148, "p": "f32", "g": "bf16",
         "copy": "bf16", "bits": 8, "step": 1000, "clip": True},
        # a table of 2^20 rows of 128, its gradient as the lookup's gradient gives it
        {"name": "adamw table 134m", "op": "adamw", "elements": 1 << 27, "tensors": 1, "p": "f32", "g": "f32", "copy": "none",
         "bits": 32, "step": 5, "clip": False},
        {"name": "adamw 8 bits table 134m", "op": "adamw", "elements": 1 << 27, "tensors": 1, "p": "f32", "g": "f32", "copy": "none",
         "bits": 8, "step": 5, "clip": False},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """1 to 2^20 rows, widths of 8 to 8192 and products of 1 to 16384 rows (half of the widths are multiples of 32, the others
    as they fall), 1000 to 2^27 elements in 1 to 200 tensors."""
    while True:
        op = rng.choice(["quant", "matmul", "matmul", "norm_matmul", "adamw", "adamw"])

        def width(lo, hi):
            k = _log_int(rng, lo, hi)
            return (k + 31) // 32 * 32 if rng.random() < 0.5 else k

        if op == "quant":
            case = {"op": op, "rows": _log_int(rng, 1, 1 << 20), "width": width(8, 8192), "x": rng.choice(["f32", "f16", "bf16"]),
                    "out": rng.choice(["f32", "f16", "bf16"])}
        elif op == "matmul":
            case = {"op": op, "m": _log_int(rng, 1, 16384), "n": width(64, 16384), "k": width(64, 8192),
                    "out": rng.choice(["f16", "bf16", "f32"]), "bias": rng.random() < 0.5}
        elif op == "norm_matmul":
            x = rng.choice(["f32", "f16", "bf16"])
            case = {"op": op, "m": _log_int(rng, 1, 1 << 20), "n": width(64, 4096), "k": width(64, 8192), "x": x,
                    "res": rng.choice(["none", x, "f16" if x == "f32" else "f32"]), "out": rng.choice(["f16", "bf16"])}
        else:
            n = _log_int(rng, 1000, 1 << 27)
            case = {"op": op, "elements": n, "tensors": min(_log_int(rng, 1, 200), n // 100), "p": rng.choice(["f32", "f32", "f32", "bf16"]),
                    "g": rng.choice(["f32", "f16", "bf16"]), "copy": rng.choice(["none", "bf16", "f16"]), "bits": rng.choice([8, 32]),
                    "step": _log_int(rng, 1, 100_000), "clip": rng.random() < 0.5}
        w = work(case)
        if w["bytes"] <= MOST_BYTES and w["flops"] <= MOST_FLOPS:
            return case


# ------------------------------------------------------------------------------------------------
# Inputs.

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(shape, dtype, gen, std=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * std).to(DTYPES[dtype])


def _uneven(shape, dtype, gen):
    """Rows as a network has them: normal values, a few channels many times as large."""
    x = torch.randn(shape, generator=gen, device="cuda")
    channel = torch.exp(0.5 * torch.randn(shape[1], generator=gen, device="cuda"))
    return x.mul_(channel).to(DTYPES[dtype])


def _blocks(k):
    return (k + BLOCK - 1) // BLOCK


def _mx4(rows, k, gen):
    """Codes [rows, 16 bytes a block], the lower half of a byte first, and scales [rows, blocks] that a program has: those
    of normal values, the last block's padding zeros."""
    blocks = _blocks(k)
    codes = torch.randint(0, 256, (rows, blocks * 16), generator=gen, device="cuda", dtype=torch.uint8)
    pad = blocks * BLOCK - k
    if pad:
        codes[:, blocks * 16 - pad // 2:] = 0
        if pad % 2:
            codes[:, blocks * 16 - pad // 2 - 1] &= 15
    scale = torch.randint(125, 129, (rows, blocks), generator=gen, device="cuda", dtype=torch.uint8)
    return codes, scale.view(torch.float8_e8m0fnu)


def _sizes(case):
    """Elements of each tensor: most of them in a few large ones."""
    rng = random.Random("%d %d" % (case["elements"], case["tensors"]))
    share = [math.exp(rng.gauss(0.0, 1.5)) for _ in range(case["tensors"])]
    sizes = [max(1, int(case["elements"] * s / sum(share))) for s in share]
    sizes[-1] = max(1, sizes[-1] + case["elements"] - sum(sizes))
    return sizes


def _adamw_inputs(case, gen):
    """Tensors as views of one flat buffer of each kind, as programs that also reduce their gradients together keep them; each
    starts on a block's boundary, what lies between is zeros."""
    sizes = _sizes(case)
    starts, total = [], 0
    for n in sizes:
        starts.append(total)
        total += _blocks(n) * BLOCK
    there = torch.zeros(total, dtype=torch.bool, device="cuda")
    for a, n in zip(starts, sizes):
        there[a:a + n] = True

    def normal(std):
        return (torch.randn(total, generator=gen, device="cuda") * std).mul_(there)

    # a quarter of the runs of 512 has had no gradient yet: rows of a table that no batch has named
    row = torch.rand((total + 511) // 512, generator=gen, device="cuda").repeat_interleave(512)[:total]
    size = torch.exp(torch.randn((total + 511) // 512, generator=gen, device="cuda")).repeat_interleave(512)[:total]
    size = size * (1e-3 * (row > 0.25))
    data = {"p": normal(0.05).to(DTYPES[case["p"]]), "g": (normal(1.0) * size).to(DTYPES[case["g"]]), "m": normal(0.3) * size,
            "v": torch.square(normal(1.0) * size * 0.7) + torch.square(0.1 * size) * there}
    if case["bits"] == 8:
        for name in ("m", "v"):
            x = data[name].view(-1, BLOCK)
            byte = ((x.abs().amax(1).view(torch.int32) >> 23) - 7).clamp(min=1)
            data[name + "_scale"] = byte.to(torch.uint8).view(torch.float8_e8m0fnu)
            x = x * ((254 - byte) << 23).view(torch.float32)[:, None]
            if name == "v":
                x = torch.where(x > 0, x.clamp(min=2.0 ** -9), x)
            data[name] = x.view(-1).to(torch.float8_e4m3fn)
    data["copy"] = None if case["copy"] == "none" else torch.zeros(total, dtype=DTYPES[case["copy"]], device="cuda")
    data["scale"] = 0.25 + 0.5 * torch.rand(1, generator=gen, device="cuda") if case["clip"] else None
    data["bounds"] = torch.tensor(starts + [total], device="cuda")
    # a norm's weights and biases, the last third of the tensors, do not decay
    return data, sizes, starts, case["tensors"] - case["tensors"] // 3


def _inputs(case, seed):
    gen, op = _gen(seed), case["op"]
    if op == "quant":
        return {"x": _uneven((case["rows"], case["width"]), case["x"], gen)}
    if op == "adamw":
        data, sizes, starts, decayed = _adamw_inputs(case, gen)
        return {**data, "sizes": sizes, "starts": starts, "decayed": decayed}
    m, n, k = case["m"], case["n"], case["k"]
    w, w_scale = _mx4(n, k, gen)
    data = {"w": w, "w_scale": w_scale}
    if op == "matmul":
        data["a"], data["a_scale"] = _mx4(m, k, gen)
        data["bias"] = _normal((n,), "f32", gen) if case["bias"] else None
        return data
    data["x"] = _uneven((m, k), case["x"], gen)
    data["res"] = None if case["res"] == "none" else _normal((m, k), case["res"], gen, 2.0)
    data["weight"] = (0.05 + 0.005 * torch.randn(k, generator=gen, device="cuda")).to(DTYPES["bf16" if case["x"] == "bf16" else "f16"])
    return data


def prepare(case, seed):
    """The tensors that a program has on the GPU before the call, and for the optimiser its lists of them."""
    state = {"case": dict(case), **_inputs(case, seed)}
    if case["op"] == "adamw":
        def views(name, per=1):
            if state.get(name) is None:
                return None
            return [state[name][a // per:a // per + (n + per - 1) // per] for a, n in zip(state["starts"], state["sizes"])]

        kinds = [views("m"), views("v")] + ([views("m_scale", BLOCK), views("v_scale", BLOCK)] if case["bits"] == 8 else [])
        state["lists"] = {"params": views("p"), "grads": views("g"), "states": list(zip(*kinds)), "copies": views("copy"),
                          "decay": [DECAY if i < state["decayed"] else 0.0 for i in range(case["tensors"])]}
    return state


# ------------------------------------------------------------------------------------------------
# The plain form: 32 bits, rounded once.

def _quantised(x):
    """The values that 4-bit codes of x [rows, width] (float32) and their block scales stand for."""
    rows, width = x.shape
    x = torch.nn.functional.pad(x, (0, _blocks(width) * BLOCK - width)).view(rows, -1, BLOCK)
    byte = ((x.abs().amax(2, keepdim=True).view(torch.int32) >> 23) - 2).clamp(min=1)
    scale = (byte << 23).view(torch.float32)
    t = x.abs() / scale
    q = torch.where(t < 2, torch.round(2 * t) / 2, torch.where(t < 4, torch.round(t), 2 * torch.round(t / 2))).clamp(max=6)
    return (torch.copysign(q, x) * scale).view(rows, -1)[:, :width]


def _values(codes, scale):
    """float32 [rows, 32 for each block] of codes and scales."""
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], device="cuda")
    q = table[torch.stack((codes & 15, codes >> 4), 2).int()].view(codes.shape[0], -1, BLOCK)
    return (q * scale.float()[:, :, None]).view(codes.shape[0], -1)


def _plain_quant(s, c):
    return _quantised(s["x"].float()).to(DTYPES[c["out"]])


def _plain_matmul(s, c):
    out = _values(s["a"], s["a_scale"]) @ _values(s["w"], s["w_scale"]).t()
    if s["bias"] is not None:
        out = out + s["bias"]
    return out.to(DTYPES[c["out"]])


def _plain_norm_matmul(s, c):
    t = s["x"].float()
    if s["res"] is not None:
        t = t + s["res"].float()
    y = _quantised(t * torch.rsqrt((t * t).mean(1, keepdim=True) + EPS) * s["weight"].float())
    out = y @ _values(s["w"], s["w_scale"])[:, :c["k"]].t()
    return {"r": None if s["res"] is None else t.to(s["res"].dtype), "out": out.to(DTYPES[c["out"]])}


def _random_bits(index, step):
    """32 bits for each element from its index in its tensor, the step's number and the seed (int64 tensors)."""
    low = 0xFFFFFFFF
    key = (SEED * 0x6A09E667 + step * 0xB7E15163) & low
    key = ((key ^ (key >> 16)) * 0xBB67AE85) & low
    x = (key + index * 0x9E3779B9 + (index >> 32) * 0x243F6A89) & low
    x = ((x ^ (x >> 15)) * 0xBB67AE85) & low
    return x ^ (x >> 16)


def _to_8_bits(x, bits):
    """x (float32) as 8-bit codes (float8_e4m3fn) and block scales; `bits`: 16 random bits for each element, which choose
    between its two neighbours."""
    x = x.view(-1, BLOCK)
    byte = ((x.abs().amax(1, keepdim=True).view(torch.int32) >> 23) - 7).clamp(min=1)
    t = x.abs() * ((254 - byte) << 23).view(torch.float32) * 2.0 ** -120   # the code is the bits' upper part
    code = (t.view(torch.int32) + (bits.view(-1, BLOCK).int() << 4) + 8) >> 20
    code = code | (x.view(torch.int32) >> 24 & 128)
    return code.to(torch.uint8).view(torch.float8_e4m3fn).view(-1), byte.to(torch.uint8).view(torch.float8_e8m0fnu).view(-1)


def _from_8_bits(codes, scale):
    return (codes.float().view(-1, BLOCK) * scale.float()[:, None]).view(-1)


def _plain_adamw(s, c):
    small = c["bits"] == 8
    g = s["g"].float()
    if s["scale"] is not None:
        g = g * s["scale"]
    m = _from_8_bits(s["m"], s["m_scale"]) if small else s["m"]
    v = _from_8_bits(s["v"], s["v_scale"]) if small else s["v"]
    m = m * BETAS[0] + g * (1 - BETAS[0])
    v = v * BETAS[1] + (g * g) * (1 - BETAS[1])
    rate, root = LR / (1 - BETAS[0] ** c["step"]), math.sqrt(1 - BETAS[1] ** c["step"])
    p = s["p"].float()
    split = s["starts"][s["decayed"]] if s["decayed"] < len(s["starts"]) else p.shape[0]
    p = torch.cat((p[:split] * (1 - LR * DECAY), p[split:])) - rate * (m / (v.sqrt() / root + ADAM_EPS))
    s["p"].copy_(p)
    if s["copy"] is not None:
        s["copy"].copy_(p)
    if small:
        first = s["bounds"][:-1].repeat_interleave(s["bounds"].diff(), output_size=p.shape[0])
        index = torch.arange(p.shape[0], device="cuda") - first
        bits = _random_bits(index, c["step"])
        s["m"], s["m_scale"] = _to_8_bits(m, bits >> 16)
        codes, s["v_scale"] = _to_8_bits(v, bits & 0xFFFF)
        # what is not zero does not become zero: the step divides by its root
        s["v"] = torch.maximum(codes.view(torch.uint8), (v > 0).to(torch.uint8)).view(torch.float8_e4m3fn)
    else:
        s["m"].copy_(m)
        s["v"].copy_(v)
    return _adamw_outputs(s)


def _adamw_outputs(s):
    return {name: s[name] for name in ("p", "m", "v", "m_scale", "v_scale", "copy") if s.get(name) is not None}


PLAIN = {"quant": _plain_quant, "matmul": _plain_matmul, "norm_matmul": _plain_norm_matmul, "adamw": _plain_adamw}


# ------------------------------------------------------------------------------------------------
# The library's calls.

_library = None


def _trspmm():
    global _library
    if _library is None:
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        sys.path.insert(0, os.path.join(root, "tr-spmm_zzx_amd"))
        import trspmm
        _library = trspmm
    return _library


def _own_quant(s, c):
    # what is held in 4 bits is compared as the values it stands for
    codes, scale = _trspmm().quant_mx4(s["x"])
    return _trspmm().dequant_mx4(codes, scale, c["width"], dtype=DTYPES[c["out"]])


def _own_matmul(s, c):
    return _trspmm().matmul_mx4(s["a"], s["a_scale"], s["w"], s["w_scale"], bias=s["bias"], dtype=DTYPES[c["out"]])


def _own_norm_matmul(s, c):
    codes, scale, r = _trspmm().rms_norm_mx4(s["x"], s["weight"], s["res"], eps=EPS)
    return {"r": r, "out": _trspmm().matmul_mx4(codes, scale, s["w"], s["w_scale"], dtype=DTYPES[c["out"]])}


def _own_adamw(s, c):
    t = s["lists"]
    _trspmm().adamw(t["params"], t["grads"], t["states"], c["step"], lr=LR, betas=BETAS, eps=ADAM_EPS, weight_decay=t["decay"],
                    copies=t["copies"], grad_scale=1.0 if s["scale"] is None else s["scale"], seed=SEED)
    return _adamw_outputs(s)


OWN = {"quant": _own_quant, "matmul": _own_matmul, "norm_matmul": _own_norm_matmul, "adamw": _own_adamw}


def run(state):
    case = state["case"]
    return (OWN if own else PLAIN)[case["op"]](state, case)


# ------------------------------------------------------------------------------------------------

def work(case):
    """quant: the rows and the values.  matmul: codes, scales, bias, output; two operations for each product.  norm_matmul:
    input, residual, weights, the new residual and the output (the codes between need not leave the chip).  adamw:
    parameters and states read and written, gradients read, copies written."""
    op = case["op"]
    if op == "quant":
        n = case["rows"] * case["width"]
        return {"bytes": n * (BYTES[case["x"]] + BYTES[case["out"]]), "flops": 6 * n}
    if op == "adamw":
        n = case["elements"]
        states = 16 if case["bits"] == 32 else 4 + 4 / BLOCK
        return {"bytes": n * (2 * BYTES[case["p"]] + BYTES[case["g"]] + BYTES[case["copy"]] + states), "flops": 16 * n}
    m, n, k = case["m"], case["n"], case["k"]
    side = _blocks(k) * 17
    if op == "matmul":
        return {"bytes": (m + n) * side + m * n * BYTES[case["out"]] + (4 * n if case["bias"] else 0), "flops": 2 * m * n * k}
    rows = m * k * (BYTES[case["x"]] + 2 * BYTES[case["res"]])
    return {"bytes": rows + 2 * k + n * side + m * n * BYTES[case["out"]], "flops": 2 * m * n * k + 6 * m * k}


# ------------------------------------------------------------------------------------------------
# The definitions in 64 bits, a slice of rows at a time.

def _slices(rows, width):
    step = max(1, (1 << 26) // max(1, width))
    return [(a, min(rows, a + step)) for a in range(0, rows, step)]


def _power(e):
    """2^e in 64 bits."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exponent(x):
    """floor(log2 x) of positive numbers, a small one for 0."""
    return torch.where(x > 0, torch.frexp(x).exponent - 1, -1000)


def _nearest4(x):
    """The 4-bit values next to x [rows, width] in 64 bits."""
    out = torch.zeros((x.shape[0], _blocks(x.shape[1]) * BLOCK), dtype=torch.float64, device="cuda")
    out[:, :x.shape[1]] = x
    blocks = out.view(x.shape[0], -1, BLOCK)
    unit = _power((_exponent(blocks.abs().max(2).values) - 2).clamp(min=-126))
    t = (blocks / unit[:, :, None]).clamp(-6.0, 6.0)
    # the distance between neighbours: 0.5 below 2, then 1, from 4 on 2
    gap = _power(_exponent(t.abs()).clamp(min=0) - 1)
    return (torch.round(t / gap) * gap * unit[:, :, None]).view(x.shape[0], -1)[:, :x.shape[1]]


def _decoded4(codes, scale):
    size = torch.tensor([0, 1, 2, 3, 4, 6, 8, 12], dtype=torch.float64, device="cuda") * 0.5
    half = torch.empty((codes.shape[0], codes.shape[1], 2), dtype=torch.float64, device="cuda")
    for i in range(2):
        c = (codes >> (4 * i)) & 15
        half[:, :, i] = size[(c & 7).long()] * (1.0 - 2.0 * (c >= 8).double())
    unit = _power(scale.view(torch.uint8).int() - 127)
    return (half.view(codes.shape[0], -1, BLOCK) * unit[:, :, None]).view(codes.shape[0], -1)


def _exact_adamw(case, d):
    n, t = d["p"].shape[0], case["step"]
    out = {name: torch.empty(n, dtype=torch.float64, device="cuda") for name in ("p", "m", "v")}
    index = torch.empty(n, dtype=torch.int64, device="cuda")
    decay = torch.zeros(n, dtype=torch.float64, device="cuda")
    ends = d["starts"][1:] + [n]
    for i, (a, b) in enumerate(zip(d["starts"], ends)):
        index[a:b] = torch.arange(b - a, device="cuda")
        decay[a:b] = DECAY if i < d["decayed"] else 0.0
    clip = 1.0 if d["scale"] is None else d["scale"].double()
    unit = {name: _power(d[name + "_scale"].view(torch.uint8).int() - 127) for name in ("m", "v")} if case["bits"] == 8 else None
    step = 1 << 24
    for a in range(0, n, step):
        b = min(n, a + step)
        g, old = d["g"][a:b].double() * clip, {name: d[name][a:b].double() for name in ("m", "v")}
        if unit:
            for name in old:
                old[name] = (old[name].view(-1, BLOCK) * unit[name][a // BLOCK:b // BLOCK, None]).view(-1)
        new = {"m": old["m"] + (1 - BETAS[0]) * (g - old["m"]), "v": old["v"] + (1 - BETAS[1]) * (g ** 2 - old["v"])}
        way = new["m"] / (1 - BETAS[0] ** t) / (torch.sqrt(new["v"] / (1 - BETAS[1] ** t)) + ADAM_EPS)
        p = d["p"][a:b].double()
        out["p"][a:b] = p - LR * decay[a:b] * p - LR * way
        if unit:
            word = _word(index[a:b], t)
            for name, chance in (("m", (word >> 16) * 16 + 8), ("v", (word % 65536) * 16 + 8)):
                x = new[name].view(-1, BLOCK)
                x = (x * _power(-(_exponent(x.abs().max(1).values) - 7).clamp(min=-126))[:, None]).view(-1)
                gap = _power(_exponent(x.abs()).clamp(min=-6) - 3)
                y = torch.floor(x.abs() / gap + chance.double() / 2 ** 20) * gap
                new[name] = torch.where(new["v"] > 0, y.clamp(min=2.0 ** -9), y) if name == "v" else torch.copysign(y, x)
        out["m"][a:b], out["v"][a:b] = new["m"], new["v"]
    out["copy"] = out["p"]
    return {name: out[name] if name in out else None for name in ("p", "m", "v", "m_scale", "v_scale", "copy") if d.get(name) is not None}


def _word(index, step):
    """The 32 bits that choose an element's rounding, one half for each of the two states."""
    mod = 1 << 32
    key = (SEED * 0x6A09E667 + step * 0xB7E15163) % mod
    key = (key ^ key // 65536) * 0xBB67AE85 % mod
    x = (index * 0x9E3779B9 + index // mod * 0x243F6A89 + key) % mod
    x = (x ^ x // 32768) * 0xBB67AE85 % mod
    return x ^ x // 65536


def exact(case, seed):
    d, op = _inputs(case, seed), case["op"]
    f64 = torch.float64
    if op == "quant":
        out = torch.empty((case["rows"], case["width"]), dtype=f64, device="cuda")
        for a, b in _slices(case["rows"], case["width"]):
            out[a:b] = _nearest4(d["x"][a:b].to(f64))
        return out
    if op == "adamw":
        return _exact_adamw(case, d)
    m, n, k = case["m"], case["n"], case["k"]
    w = _decoded4(d["w"], d["w_scale"])[:, :k].t().contiguous()
    out = torch.empty((m, n), dtype=f64, device="cuda")
    if op == "matmul":
        for a, b in _slices(m, max(n, k)):
            out[a:b] = torch.mm(_decoded4(d["a"][a:b], d["a_scale"][a:b])[:, :k], w)
        return out if d["bias"] is None else out.add_(d["bias"].to(f64))
    has = d["res"] is not None
    r = torch.empty((m, k), dtype=f64, device="cuda") if has else None
    for a, b in _slices(m, max(n, k)):
        h = d["x"][a:b].to(f64) + (d["res"][a:b].to(f64) if has else 0.0)
        if has:
            r[a:b] = h
        length = torch.linalg.vector_norm(h, dim=1, keepdim=True)
        out[a:b] = torch.mm(_nearest4(h / torch.sqrt(length * length / k + EPS) * d["weight"].to(f64)), w)
    return {"r": r, "out": out}
