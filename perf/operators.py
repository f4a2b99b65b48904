"""The dense operators beside the sparse products, as measurable cases: what a layer of a graph model does to the
features before and after ``Plan.spmm``.

A case is a plain dict:

    op      "embed"       rows of a node or token table for a batch of ids, times a scale
            "embed_grad"  its gradient: the gradients of equal ids summed into the table's rows, zeros elsewhere
            "norm"        root-mean-square norm of x (+ residual): the new residual and, by `out`, the normed rows in
                          8 bits with a scale for each row ("i8") or in 16 or 32 bits
            "norm_grad"   the norm's gradient: towards its input (the residual's own gradient added) and its weight
            "matmul"      codes in 8 bits times weights in 8 bits, with a scale for each row and each output channel
    rows, count, width    table rows, ids, features                                           (embed, embed_grad)
    skew, pad             how far the ids lean to few rows (1 = even), share of ids that are -1 (padded slots)
    tokens, width         rows and features                                                   (norm, norm_grad)
    m, n, k               rows, output channels, inner length                                 (matmul)
    x, res, out           types of the input, the residual ("none" without one) and the output

Where `own` is false, `run` computes the same in elementary torch operations in 32 bits.
"""
import math
import os
import sys

import torch

#: Set by who measures: true for the library's kernels, false for the plain form.
own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2, "i8": 1, "none": 0}
EPS = 1e-5

#: What the largest listed cases cost: no drawn case has more of either.
MOST_BYTES = 900_000_000
MOST_FLOPS = 2 * 8192 ** 3


def listed():
    return [
        # the nodes of one small sampled neighbourhood: latency
        {"name": "embed 256 of 64k d128", "op": "embed", "rows": 1 << 16, "count": 256, "width": 128, "skew": 1, "pad": 0.0,
         "bits": 64, "x": "f16", "out": "f16", "scale": 1.0},
        # all slots of a large sampled batch out of the headline graph's 2^20 nodes, hubs more often, some slots padded
        {"name": "embed 1m of 1m d128", "op": "embed", "rows": 1 << 20, "count": 1_000_003, "width": 128, "skew": 2, "pad": 0.02,
         "bits": 32, "x": "f16", "out": "f16", "scale": 11.3137085},
        # the gradient of a mini-batch into a small table
        {"name": "embed_grad 4k into 16k d64", "op": "embed_grad", "rows": 1 << 14, "count": 4096, "width": 64, "skew": 2, "pad": 0.02,
         "bits": 64, "x": "f16", "out": "f32", "scale": 8.0},
        # the gradient of the large batch: the most frequent id comes thousands of times
        {"name": "embed_grad 1m into 1m d128", "op": "embed_grad", "rows": 1 << 20, "count": 1_000_003, "width": 128, "skew": 3,
         "pad": 0.02, "bits": 32, "x": "f16", "out": "f32", "scale": 11.3137085},
        # serving, one token: the residual's addition, the norm and its 8-bit codes
        {"name": "norm i8 1 x 4096", "op": "norm", "tokens": 1, "width": 4096, "x": "f16", "res": "f16", "out": "i8"},
        # what an aggregation hands on: float32 sums of 2^20 nodes, hidden width 128, residual in 16 bits
        {"name": "norm i8 1m x 128", "op": "norm", "tokens": 1 << 20, "width": 128, "x": "f32", "res": "f16", "out": "i8"},
        # training or prefill: 16 bits in and out
        {"name": "norm bf16 16k x 4096", "op": "norm", "tokens": 16384, "width": 4096, "x": "bf16", "res": "bf16", "out": "bf16"},
        # the gradient at an odd number of rows and a width off the power of two
        {"name": "norm_grad 4099 x 1000", "op": "norm_grad", "tokens": 4099, "width": 1000, "x": "f16"},
        # the gradient of a training step
        {"name": "norm_grad 16k x 4096", "op": "norm_grad", "tokens": 16384, "width": 4096, "x": "bf16"},
        # serving, one token: bound by the weights
        {"name": "matmul 1 x 4096 x 4096", "op": "matmul", "m": 1, "n": 4096, "k": 4096, "out": "f16", "bias": False},
        # a layer's projection over all nodes, hidden width 128 to 256: bound by the rows
        {"name": "matmul 1m x 256 x 128", "op": "matmul", "m": 1_000_003, "n": 256, "k": 128, "out": "f16", "bias": True},
        # a large batch through a wide layer: bound by arithmetic
        {"name": "matmul 8k x 8k x 8k", "op": "matmul", "m": 8192, "n": 8192, "k": 8192, "out": "bf16", "bias": False},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """Tables of 1024 to 2^20 rows, 1 to 2^20 ids or rows, widths of 8 to 8192, products of 1 to 16384 rows; half of the
    widths are multiples of 8, the others as they fall."""
    while True:
        op = rng.choice(["embed", "embed_grad", "norm", "norm_grad", "matmul", "matmul"])

        def width(lo, hi):
            k = _log_int(rng, lo, hi)
            return (k + 7) // 8 * 8 if rng.random() < 0.5 else k

        if op in ("embed", "embed_grad"):
            case = {"op": op, "rows": _log_int(rng, 1024, 1 << 20), "count": _log_int(rng, 1, 1 << 20), "width": width(8, 1024),
                    "skew": rng.choice([1, 2, 3]), "pad": rng.choice([0.0, 0.02, 0.2]), "bits": rng.choice([32, 64]),
                    "x": rng.choice(["f32", "f16", "bf16"]), "scale": round(rng.uniform(0.5, 12.0), 3)}
            case["out"] = rng.choice([case["x"], "f32"])
        elif op == "norm":
            case = {"op": op, "tokens": _log_int(rng, 1, 1 << 20), "width": width(64, 8192), "x": rng.choice(["f32", "f16", "bf16"])}
            case["res"] = rng.choice(["none", case["x"], "f16" if case["x"] == "f32" else "f32"])
            case["out"] = rng.choice(["i8", "i8", "bf16" if case["x"] == "bf16" else "f16"])
        elif op == "norm_grad":
            case = {"op": op, "tokens": _log_int(rng, 1, 1 << 20), "width": width(64, 8192), "x": rng.choice(["f32", "f16", "bf16"])}
        else:
            case = {"op": op, "m": _log_int(rng, 1, 16384), "n": width(64, 16384), "k": width(64, 8192),
                    "out": rng.choice(["f16", "bf16", "f32"]), "bias": rng.random() < 0.5}
        w = work(case)
        if w["bytes"] <= MOST_BYTES and w["flops"] <= MOST_FLOPS:
            return case


# ------------------------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(shape, dtype, gen, std=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * std).to(DTYPES[dtype])


def _ids(case, gen):
    """Ids that lean to few rows, which lie anywhere in the table; -1 for padded slots."""
    rows, count = case["rows"], case["count"]
    rank = (torch.rand(count, generator=gen, device="cuda", dtype=torch.float64) ** case["skew"] * rows).long().clamp(max=rows - 1)
    ids = torch.randperm(rows, generator=gen, device="cuda")[rank]
    ids = torch.where(torch.rand(count, generator=gen, device="cuda") < case["pad"], -1, ids)
    return ids.to(torch.int32 if case["bits"] == 32 else torch.int64)


def _codes(rows, width, gen):
    return torch.randint(-127, 128, (rows, width), generator=gen, device="cuda", dtype=torch.int8)


def _scales(count, width, gen):
    """Scales that bring a product of `width` codes near 1."""
    return (0.5 + torch.rand(count, generator=gen, device="cuda")) / (73.0 * math.sqrt(math.sqrt(width)))


def _inputs(case, seed):
    gen, op = _gen(seed), case["op"]
    if op in ("embed", "embed_grad"):
        shape = (case["rows" if op == "embed" else "count"], case["width"])
        return {"ids": _ids(case, gen), "x": _normal(shape, case["x"], gen, 0.1)}
    if op in ("norm", "norm_grad"):
        t, d, x = case["tokens"], case["width"], case["x"]
        small = "bf16" if x == "bf16" else "f16"
        data = {"weight": (1 + 0.1 * torch.randn(d, generator=gen, device="cuda")).to(DTYPES[small])}
        if op == "norm":
            data["x"] = _normal((t, d), x, gen)
            data["res"] = None if case["res"] == "none" else _normal((t, d), case["res"], gen, 2.0)
        else:
            data["r"] = _normal((t, d), x, gen, 2.0)
            data["grad"] = _normal((t, d), x, gen, 0.1)
            data["grad_r"] = _normal((t, d), x, gen, 0.1)
        return data
    m, n, k = case["m"], case["n"], case["k"]
    return {"a": _codes(m, k, gen), "w": _codes(n, k, gen), "a_scale": _scales(m, k, gen), "w_scale": _scales(n, k, gen),
            "bias": _normal((n,), "f32", gen) if case["bias"] else None}


def prepare(case, seed):
    """The tensors that a program has on the GPU before the call; the operators keep no plan."""
    return {"case": dict(case), **_inputs(case, seed)}


# ------------------------------------------------------------------------------------------------
# The plain form: 32 bits, rounded once.

def _plain_embed(s, c):
    ids = s["ids"].long()
    rows = s["x"][ids.clamp(min=0)].float() * c["scale"]
    return rows.masked_fill_((ids < 0)[:, None], 0.0).to(DTYPES[c["out"]])


def _plain_embed_grad(s, c):
    rows = c["rows"]
    ids = s["ids"].long()
    total = torch.zeros((rows + 1, c["width"]), device="cuda")
    total.index_add_(0, torch.where(ids < 0, rows, ids), s["x"].float())
    return (total[:rows] * c["scale"]).to(DTYPES[c["out"]])


def _plain_norm(s, c):
    t = s["x"].float()
    if s["res"] is not None:
        t = t + s["res"].float()
    y = t * torch.rsqrt((t * t).mean(1, keepdim=True) + EPS) * s["weight"].float()
    r = None if s["res"] is None else t.to(s["res"].dtype)
    if c["out"] != "i8":
        return {"y": y.to(DTYPES[c["out"]]), "r": r}
    scale = y.abs().amax(1, keepdim=True) / 127
    codes = torch.where(scale > 0, torch.round(y / scale), 0.0)
    return {"y": (codes * scale).to(s["weight"].dtype), "r": r}


def _plain_norm_grad(s, c):
    r, grad = s["r"].float(), s["grad"].float()
    rstd = torch.rsqrt((r * r).mean(1, keepdim=True) + EPS)
    unit = r * rstd
    g = grad * s["weight"].float()
    dr = rstd * (g - unit * (g * unit).mean(1, keepdim=True)) + s["grad_r"].float()
    return {"r": dr.to(s["r"].dtype), "weight": (grad * unit).sum(0)}


def _plain_matmul(s, c):
    out = s["a"].float() @ s["w"].float().t()
    out = out * s["a_scale"][:, None] * s["w_scale"]
    if s["bias"] is not None:
        out = out + s["bias"]
    return out.to(DTYPES[c["out"]])


PLAIN = {"embed": _plain_embed, "embed_grad": _plain_embed_grad, "norm": _plain_norm, "norm_grad": _plain_norm_grad,
         "matmul": _plain_matmul}


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


def _own_embed(s, c):
    return _trspmm().embed(s["x"], s["ids"], scale=c["scale"], dtype=DTYPES[c["out"]])


def _own_embed_grad(s, c):
    return _trspmm().embed_grad(s["x"], s["ids"], c["rows"], scale=c["scale"], dtype=DTYPES[c["out"]])


def _own_norm(s, c):
    if c["out"] != "i8":
        y, r = _trspmm().rms_norm(s["x"], s["weight"], s["res"], eps=EPS, dtype=DTYPES[c["out"]])
        return {"y": y, "r": r}
    codes, scale, r = _trspmm().rms_norm_i8(s["x"], s["weight"], s["res"], eps=EPS)
    # what is held in 8 bits is compared as the values it stands for
    y = torch.empty(codes.shape, dtype=s["weight"].dtype, device="cuda")
    return {"y": torch.mul(codes, scale[:, None], out=y), "r": r}


def _own_norm_grad(s, c):
    dr, dweight = _trspmm().rms_norm_grad(s["grad"], s["r"], s["weight"], s["grad_r"], eps=EPS)
    return {"r": dr, "weight": dweight}


def _own_matmul(s, c):
    return _trspmm().matmul_i8(s["a"], s["a_scale"], s["w"], s["w_scale"], bias=s["bias"], dtype=DTYPES[c["out"]])


OWN = {"embed": _own_embed, "embed_grad": _own_embed_grad, "norm": _own_norm, "norm_grad": _own_norm_grad,
       "matmul": _own_matmul}


def run(state):
    case = state["case"]
    return (OWN if own else PLAIN)[case["op"]](state, case)


# ------------------------------------------------------------------------------------------------

def work(case):
    """embed: the ids, the table rows that can differ, the output.  embed_grad: the ids, the gradients, the whole table's
    gradient.  norm: x, residual, weight, the new residual and the normed rows, each once ("i8": codes and scales).
    norm_grad: three inputs and one output of the rows' size, the weight and its gradient.  matmul: codes, scales, output;
    two operations for each product."""
    op = case["op"]
    if op in ("embed", "embed_grad"):
        count, rows, d = case["count"], case["rows"], case["width"]
        x, out = BYTES[case["x"]], BYTES[case["out"]]
        if op == "embed":
            return {"bytes": count * case["bits"] // 8 + min(count, rows) * d * x + count * d * out, "flops": count * d}
        return {"bytes": count * case["bits"] // 8 + count * d * x + rows * d * out, "flops": 2 * count * d}
    if op in ("norm", "norm_grad"):
        t, d, x = case["tokens"], case["width"], BYTES[case["x"]]
        if op == "norm":
            rows = t * d * (x + 2 * BYTES[case["res"]] + BYTES[case["out"]])
            return {"bytes": rows + 2 * d + (4 * t if case["out"] == "i8" else 0), "flops": 6 * t * d}
        return {"bytes": 4 * t * d * x + 6 * d, "flops": 12 * t * d}
    m, n, k = case["m"], case["n"], case["k"]
    return {"bytes": m * k + n * k + 4 * (m + n) + m * n * BYTES[case["out"]], "flops": 2 * m * n * k}


# ------------------------------------------------------------------------------------------------
# The definitions in 64 bits, a slice of rows at a time.

def _slices(rows, width):
    step = max(1, (1 << 26) // max(1, width))
    return [(a, min(rows, a + step)) for a in range(0, rows, step)]


def exact(case, seed):
    d, op = _inputs(case, seed), case["op"]
    f64 = torch.float64
    if op == "embed":
        out = torch.zeros((case["count"], case["width"]), dtype=f64, device="cuda")
        there = torch.nonzero(d["ids"] >= 0).flatten()
        for a, b in _slices(there.shape[0], case["width"]):
            out[there[a:b]] = d["x"].index_select(0, d["ids"][there[a:b]].int()).to(f64) * case["scale"]
        return out
    if op == "embed_grad":
        out = torch.zeros((case["rows"], case["width"]), dtype=f64, device="cuda")
        there = torch.nonzero(d["ids"] >= 0).flatten()
        for a, b in _slices(there.shape[0], case["width"]):
            out.index_add_(0, d["ids"][there[a:b]].int(), d["x"][there[a:b]].to(f64) * case["scale"])
        return out
    if op == "norm":
        has = d["res"] is not None
        y = torch.empty((case["tokens"], case["width"]), dtype=f64, device="cuda")
        r = torch.empty_like(y) if has else None
        for a, b in _slices(case["tokens"], case["width"]):
            h = d["x"][a:b].to(f64) + (d["res"][a:b].to(f64) if has else 0.0)
            if has:
                r[a:b] = h
            length = torch.linalg.vector_norm(h, dim=1, keepdim=True)
            v = h / torch.sqrt(length * length / case["width"] + EPS) * d["weight"].to(f64)
            if case["out"] == "i8":
                unit = v.abs().max(1, keepdim=True).values / 127.0
                v = torch.round(v / unit.clamp(min=1e-300)) * unit
            y[a:b] = v
        return {"y": y, "r": r}
    if op == "norm_grad":
        dr = torch.empty((case["tokens"], case["width"]), dtype=f64, device="cuda")
        dw = torch.zeros(case["width"], dtype=f64, device="cuda")
        w = d["weight"].to(f64)
        for a, b in _slices(case["tokens"], case["width"]):
            h, g = d["r"][a:b].to(f64), d["grad"][a:b].to(f64)
            inv = 1.0 / torch.sqrt((h ** 2).sum(1) / case["width"] + EPS)
            dot = (g * w * h).sum(1)
            dr[a:b] = g * w * inv[:, None] - h * (inv ** 3 * dot / case["width"])[:, None] + d["grad_r"][a:b].to(f64)
            dw += (g * h * inv[:, None]).sum(0)
        return {"r": dr, "weight": dw}
    out = torch.empty((case["m"], case["n"]), dtype=f64, device="cuda")
    w = d["w"].to(f64).t().contiguous()
    for a, b in _slices(case["m"], max(case["n"], case["k"])):
        out[a:b] = torch.mm(d["a"][a:b].to(f64), w)
        out[a:b] *= torch.outer(d["a_scale"][a:b].to(f64), d["w_scale"].to(f64))
        if d["bias"] is not None:
            out[a:b] += d["bias"].to(f64)
    return out
