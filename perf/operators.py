"""Cases, plain forms and calls of the low-precision and grouped products.

  quantize       a matrix as 8-bit floating point (e4m3) with a power-of-two scale for each block of 128
  linear_fp8     y = act(x W^T + b) on such operands, and `linear_fp8_grad`, the gradient of its input
  grouped        products of ragged row groups, each with a weight of its own, and `grouped_grad`, their backward pass
  saved          the backward pass of act(x W^T + b) from x and the pre-activation kept in 8 bits

Sizes: the Linear stack of the benchmark (8192 rows, 4096 -> 16384 -> 4096), its small-batch forms, and expert
layers of the same widths.
"""
import ctypes
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODES = {"f32": 0, "f16": 1, "bf16": 2}
ACTS = {"none": 0, "relu": 1, "gelu": 2, "silu": 3, "sigmoid": 4}
BLOCK = 128
MOST_QUANTIZE = 8192 * 16384
MOST_LINEAR = 8192 * 16384 * 4096
MOST_GROUPED = 16384 * 4096 * 2048
MOST_WEIGHTS = 32 * 4096 * 2048
MOST_SAVED = 8192 * 4096 * 4096


def listed():
    return [
        # the activations of eight sequences that each decode one token
        {"name": "quantize_decode", "op": "quantize", "type": "bf16", "rows": 8, "cols": 4096, "block_rows": 1},
        # the hidden activation of the Linear stack, kept for its backward pass
        {"name": "quantize_hidden", "op": "quantize", "type": "bf16", "rows": 8192, "cols": 16384, "block_rows": 1},
        # a single-precision weight whose sides are no multiples of the block, prepared once or after each update
        {"name": "quantize_weight", "op": "quantize", "type": "f32", "rows": 4100, "cols": 11007, "block_rows": 128},
        # the stack's first layer for sixteen tokens: the weight's bytes are what it costs
        {"name": "linear_decode", "op": "linear_fp8", "type": "bf16", "m": 16, "n": 16384, "k": 4096, "act": "none",
         "bias": False},
        # the stack's first layer with its bias and activation
        {"name": "linear_layer", "op": "linear_fp8", "type": "bf16", "m": 8192, "n": 16384, "k": 4096, "act": "gelu",
         "bias": True},
        # the gradient of the input of a layer with odd sides for a ragged batch, kept in single precision
        {"name": "linear_grad_ragged", "op": "linear_fp8_grad", "type": "f32", "m": 2047, "n": 5000, "k": 1672},
        # experts that decode: a few rows each, some none
        {"name": "grouped_decode", "op": "grouped", "type": "bf16", "rows": 64, "groups": 16, "n": 4096, "k": 1024},
        # an expert layer of a training batch, with padding rows behind the last group
        {"name": "grouped_layer", "op": "grouped", "type": "bf16", "rows": 16384, "groups": 32, "n": 4096, "k": 2048},
        # odd widths, few uneven groups
        {"name": "grouped_ragged", "op": "grouped", "type": "f16", "rows": 1537, "groups": 5, "n": 777, "k": 1001},
        # the backward pass of an expert layer: gradient of the rows, and of the weights in single precision
        {"name": "grouped_grad", "op": "grouped_grad", "type": "bf16", "grad_type": "f32", "rows": 8192, "groups": 16,
         "n": 2048, "k": 2048},
        # a layer's backward pass from what was kept in 8 bits
        {"name": "saved_layer", "op": "saved", "type": "bf16", "m": 8192, "n": 4096, "k": 4096, "act": "gelu"},
        # the same for a short batch and odd widths
        {"name": "saved_ragged", "op": "saved", "type": "f16", "m": 333, "n": 520, "k": 1023, "act": "silu"},
    ]


def _size(rng, low, high):
    s = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    step = rng.choice([1, 1, 2, 8, 16, 128])
    if s >= 4 * step:
        s -= s % step
    return max(low, min(high, s))


def draw(rng):
    op = rng.choice(["quantize", "linear_fp8", "linear_fp8", "linear_fp8_grad", "grouped", "grouped", "grouped_grad",
                     "saved"])
    half = rng.choice(["f16", "bf16"])
    while True:
        if op == "quantize":
            c = {"op": op, "type": rng.choice(["f32", half]), "rows": _size(rng, 1, 16384),
                 "cols": _size(rng, 64, 16384), "block_rows": rng.choice([1, 128])}
            if c["rows"] * c["cols"] <= MOST_QUANTIZE // 2:
                return c
        elif op in ("linear_fp8", "linear_fp8_grad"):
            c = {"op": op, "type": rng.choice(["f32", half]), "m": _size(rng, 1, 8192), "n": _size(rng, 64, 16384),
                 "k": _size(rng, 64, 16384)}
            if op == "linear_fp8":
                c["act"] = rng.choice(sorted(ACTS))
                c["bias"] = rng.random() < 0.5
            if c["m"] * c["n"] * c["k"] <= MOST_LINEAR:
                return c
        elif op in ("grouped", "grouped_grad"):
            c = {"op": op, "type": half, "rows": _size(rng, 1, 16384), "groups": _size(rng, 1, 64),
                 "n": _size(rng, 64, 4096), "k": _size(rng, 64, 4096)}
            if op == "grouped_grad":
                c["grad_type"] = rng.choice(["f32", half])
            if (c["rows"] * c["n"] * c["k"] * (3 if op == "grouped_grad" else 1) <= MOST_GROUPED
                    and c["groups"] * c["n"] * c["k"] <= MOST_WEIGHTS):
                return c
        else:
            c = {"op": op, "type": half, "m": _size(rng, 1, 8192), "n": _size(rng, 64, 4096),
                 "k": _size(rng, 64, 4096), "act": rng.choice(sorted(ACTS))}
            if c["m"] * c["n"] * c["k"] <= MOST_SAVED:
                return c


# ---- inputs ------------------------------------------------------------------------------------------------


def _normal(gen, shape, dtype, std=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * std).to(dtype)


def _weight(gen, shape, dtype):
    bound = math.sqrt(6.0 / shape[-1])
    return ((torch.rand(shape, generator=gen, device="cuda") * 2 - 1) * bound).to(dtype)


def _activations(gen, rows, cols, dtype):
    """Rows of different sizes with a few columns that stand out, as activations have."""
    x = torch.randn(rows, cols, generator=gen, device="cuda")
    x *= torch.exp(torch.randn(rows, 1, generator=gen, device="cuda") * 0.5)
    x *= torch.where(torch.rand(1, cols, generator=gen, device="cuda") < 0.01, 20.0, 1.0)
    return x.to(dtype)


def _group_sizes(case, seed):
    """Uneven sizes, some of them zero, of up to all rows; what is left over is padding behind the last group."""
    rng = random.Random(seed * 7919 + 17)
    groups, rows = case["groups"], case["rows"]
    used = rows - (rng.randrange(rows // 16 + 1) if rows > 16 else 0)
    share = [rng.gammavariate(3.0, 1.0) * (rng.random() >= 0.05) for _ in range(groups)]
    if not sum(share):
        share[-1] = 1.0
    cuts, acc = [0], 0.0
    for s in share:
        acc += s
        cuts.append(int(round(used * acc / sum(share))))
    return [b - a for a, b in zip(cuts, cuts[1:])]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed) + 1)
    op, t = case["op"], TYPES[case["type"]]
    s = {"case": case}
    if op == "quantize":
        rows, cols = case["rows"], case["cols"]
        if case["block_rows"] == 1:
            s["x"] = _activations(gen, rows, cols, t)
            s["scales"] = torch.empty(-(-cols // BLOCK), rows, device="cuda")
        else:
            s["x"] = _weight(gen, (rows, cols), t)
            s["scales"] = torch.empty(-(-rows // BLOCK), -(-cols // BLOCK), device="cuda")
        s["q"] = torch.empty(rows, cols, dtype=torch.uint8, device="cuda")
    elif op in ("linear_fp8", "linear_fp8_grad"):
        m, n, k = case["m"], case["n"], case["k"]
        inner, outer = (k, n) if op == "linear_fp8" else (n, k)
        s["x8"], s["xs"] = _quantize(_activations(gen, m, inner, torch.float32), 1)
        s["w8"], s["ws"] = _quantize(_weight(gen, (n, k), torch.float32), BLOCK)
        s["bias"] = _normal(gen, (n,), torch.float32, 0.5) if case.get("bias") else None
        s["y"] = torch.zeros(m, outer, dtype=t, device="cuda")
    elif op in ("grouped", "grouped_grad"):
        sizes = _group_sizes(case, seed)
        s["sizes"] = sizes
        s["most"] = max(sizes)
        s["offsets"] = torch.tensor([sum(sizes[:i]) for i in range(len(sizes) + 1)], dtype=torch.int32, device="cuda")
        rows, groups, n, k = case["rows"], case["groups"], case["n"], case["k"]
        s["x"] = _normal(gen, (rows, k), t)
        s["w"] = _weight(gen, (groups, n, k), t)
        if op == "grouped":
            s["y"] = torch.zeros(rows, n, dtype=t, device="cuda")
        else:
            s["dy"] = _normal(gen, (rows, n), t, 0.1)
            s["dx"] = torch.zeros(rows, k, dtype=t, device="cuda")
            s["dw"] = torch.zeros(groups, n, k, dtype=TYPES[case["grad_type"]], device="cuda")
    else:
        m, n, k = case["m"], case["n"], case["k"]
        s["x8"], s["xs"] = _quantize(_activations(gen, m, k, torch.float32), 1)
        s["z8"], s["zs"] = _quantize(_normal(gen, (m, n), torch.float32, 1.5), 1)
        s["w"] = _weight(gen, (n, k), t)
        s["dy"] = _normal(gen, (m, n), t, 0.1)
        s["dx"] = torch.zeros(m, k, dtype=t, device="cuda")
        s["dw"] = torch.zeros(n, k, dtype=t, device="cuda")
        s["db"] = torch.zeros(n, device="cuda")
    return s


# ---- the plain forms ---------------------------------------------------------------------------------------


def _power_of_two_scale(amax):
    """The smallest power of two (2^-126 at least, 1 for a block of zeros) under which amax / scale <= 448."""
    mantissa, exponent = torch.frexp(amax)                 # amax = mantissa * 2^exponent, mantissa in [0.5, 1)
    exponent = (exponent - 9 + (mantissa > 0.875)).clamp(min=-126)
    return torch.where(amax == 0, torch.ones_like(amax), torch.ldexp(torch.ones_like(amax), exponent))


def _quantize(x, block_rows):
    """e4m3 values and scales: [blocks of columns, rows] for blocks of 1 x 128, [blocks of rows, blocks of columns]
    for blocks of 128 x 128."""
    rows, cols = x.shape
    cb, rb = -(-cols // BLOCK), -(-rows // block_rows)
    p = torch.zeros(rb * block_rows, cb * BLOCK, device=x.device)
    p[:rows, :cols] = x
    p = p.view(rb, block_rows, cb, BLOCK)
    amax = torch.where(torch.isfinite(p), p.abs(), torch.zeros_like(p)).amax(dim=(1, 3), keepdim=True)
    scale = _power_of_two_scale(amax)
    p = (p / scale).view(rb * block_rows, cb * BLOCK)[:rows, :cols]
    q = torch.where(torch.isfinite(p), p, torch.full_like(p, math.nan)).to(torch.float8_e4m3fn)
    scale = scale.view(rb, cb)
    return q, (scale.t().contiguous() if block_rows == 1 else scale)


def _rows_value(q, scales):
    """What blocks of 1 x 128 stand for, in 32 bits."""
    cols = q.shape[1]
    return q.float() * scales.t().repeat_interleave(BLOCK, dim=1)[:, :cols]


def _tiles_value(q, scales):
    rows, cols = q.shape
    return q.float() * scales.repeat_interleave(BLOCK, dim=0)[:rows].repeat_interleave(BLOCK, dim=1)[:, :cols]


def _act(z, name):
    if name == "relu":
        return z.clamp(min=0)
    if name == "gelu":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    if name == "silu":
        return z / (1 + torch.exp(-z))
    if name == "sigmoid":
        return 1 / (1 + torch.exp(-z))
    return z


def _act_slope(z, name):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "gelu":
        c = math.sqrt(2 / math.pi)
        th = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + th) + 0.5 * z * (1 - th * th) * c * (1 + 3 * 0.044715 * z * z)
    s = 1 / (1 + torch.exp(-z))
    if name == "silu":
        return s * (1 + z * (1 - s))
    if name == "sigmoid":
        return s * (1 - s)
    return torch.ones_like(z)


def _padded(x, s):
    """[groups, rows of the largest group, columns] in 32 bits, zeros behind each group's rows, and where they lie."""
    at = s["offsets"][:-1, None] + torch.arange(s["most"], device="cuda")[None]
    real = at < s["offsets"][1:, None]
    at = at.clamp(max=x.shape[0] - 1).long()
    return torch.where(real[..., None], x[at].float(), 0.0), at, real


def _plain(s):
    case = s["case"]
    op, t = case["op"], TYPES[case["type"]]
    if op == "quantize":
        return _quantize(s["x"].float(), case["block_rows"])
    if op == "linear_fp8":
        y = _rows_value(s["x8"], s["xs"]) @ _tiles_value(s["w8"], s["ws"]).t()
        if s["bias"] is not None:
            y = y + s["bias"]
        return _act(y, case["act"]).to(t)
    if op == "linear_fp8_grad":
        return (_rows_value(s["x8"], s["xs"]) @ _tiles_value(s["w8"], s["ws"])).to(t)
    if op == "grouped":
        x, at, real = _padded(s["x"], s)
        y = torch.bmm(x, s["w"].float().transpose(1, 2)).to(t)
        out = torch.zeros(case["rows"], case["n"], dtype=t, device="cuda")
        out[at[real]] = y[real]
        return out
    if op == "grouped_grad":
        x, at, real = _padded(s["x"], s)
        dy, _, _ = _padded(s["dy"], s)
        g = torch.bmm(dy, s["w"].float()).to(t)
        dx = torch.zeros(case["rows"], case["k"], dtype=t, device="cuda")
        dx[at[real]] = g[real]
        return dx, torch.bmm(dy.transpose(1, 2), x).to(TYPES[case["grad_type"]])
    z = _rows_value(s["z8"], s["zs"])
    dz = s["dy"].float() * _act_slope(z, case["act"])
    return (dz @ s["w"].float()).to(t), (dz.t() @ _rows_value(s["x8"], s["xs"])).to(t), dz.sum(0)


# ---- the framework's calls -----------------------------------------------------------------------------------


def _p(t):
    return None if t is None else t.data_ptr()


def _own(s):
    from cudeep_b200 import _lib

    lib, case = _lib.load(), s["case"]
    op, code = case["op"], CODES[case["type"]]
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    if op == "quantize":
        _lib.check(lib.cudeep_b200_quantize_fp8(_p(s["x"]), code, case["rows"], case["cols"], case["block_rows"],
                                                _p(s["q"]), _p(s["scales"]), stream))
        return s["q"].view(torch.float8_e4m3fn), s["scales"]
    if op == "linear_fp8":
        _lib.check(lib.cudeep_b200_linear_forward_fp8(_p(s["x8"]), _p(s["xs"]), _p(s["w8"]), _p(s["ws"]),
                                                      _p(s["bias"]), _p(s["y"]), code, case["m"], case["n"], case["k"],
                                                      ACTS[case["act"]], stream))
        return s["y"]
    if op == "linear_fp8_grad":
        _lib.check(lib.cudeep_b200_linear_backward_data_fp8(_p(s["x8"]), _p(s["xs"]), _p(s["w8"]), _p(s["ws"]),
                                                            _p(s["y"]), code, case["m"], case["n"], case["k"], stream))
        return s["y"]
    if op == "grouped":
        _lib.check(lib.cudeep_b200_grouped_matmul_nt(_p(s["x"]), _p(s["w"]), _p(s["y"]), code, _p(s["offsets"]),
                                                     case["groups"], case["rows"], case["n"], case["k"], stream))
        return s["y"]
    if op == "grouped_grad":
        _lib.check(lib.cudeep_b200_grouped_matmul_nn(_p(s["dy"]), _p(s["w"]), _p(s["dx"]), code, _p(s["offsets"]),
                                                     case["groups"], case["rows"], case["k"], case["n"], stream))
        _lib.check(lib.cudeep_b200_grouped_matmul_tn(_p(s["dy"]), _p(s["x"]), _p(s["dw"]), code,
                                                     CODES[case["grad_type"]], _p(s["offsets"]), case["groups"],
                                                     case["rows"], case["n"], case["k"], stream))
        return s["dx"], s["dw"]
    _lib.check(lib.cudeep_b200_linear_backward_saved_fp8(
        _p(s["dy"]), code, _p(s["x8"]), _p(s["xs"]), _p(s["z8"]), _p(s["zs"]), ACTS[case["act"]], _p(s["w"]),
        _p(s["dx"]), _p(s["dw"]), code, _p(s["db"]), case["m"], case["n"], case["k"], stream))
    return s["dx"], s["dw"], s["db"]


def run(state):
    return _own(state) if own else _plain(state)


# ---- work and exact values -----------------------------------------------------------------------------------


def work(case):
    op = case["op"]
    size = {"f32": 4, "f16": 2, "bf16": 2}
    b = size[case["type"]]
    if op == "quantize":
        rows, cols = case["rows"], case["cols"]
        blocks = -(-rows // case["block_rows"]) * -(-cols // BLOCK)
        return {"bytes": rows * cols * (b + 1) + 4 * blocks, "flops": 2 * rows * cols}
    if op in ("linear_fp8", "linear_fp8_grad"):
        m, n, k = case["m"], case["n"], case["k"]
        inner, outer = (k, n) if op == "linear_fp8" else (n, k)
        scales = 4 * (m * -(-inner // BLOCK) + -(-n // BLOCK) * -(-k // BLOCK))
        return {"bytes": m * inner + n * k + scales + b * m * outer + (4 * n if case.get("bias") else 0),
                "flops": 2 * m * n * k}
    if op in ("grouped", "grouped_grad"):
        rows, n, k = case["rows"], case["n"], case["k"]
        used = min(case["groups"], rows)
        if op == "grouped":
            return {"bytes": b * (rows * k + used * n * k + rows * n), "flops": 2 * rows * n * k}
        return {"bytes": b * (2 * rows * k + used * n * k + rows * n) + size[case["grad_type"]] * case["groups"] * n * k,
                "flops": 4 * rows * n * k}
    m, n, k = case["m"], case["n"], case["k"]
    scales = 4 * m * (-(-k // BLOCK) + -(-n // BLOCK))
    return {"bytes": b * (m * n + 2 * n * k + m * k) + m * k + m * n + scales + 4 * n, "flops": 4 * m * n * k}


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    wide = torch.float64
    if op == "quantize":
        # Whole by whole: the scale from the binary logarithm's floor, corrected by comparison; the values are the
        # type's own, so only the scales are numbers in 64 bits.
        x = s["x"].to(wide).abs()
        cols = x.shape[1]
        parts = [x[:, c:c + BLOCK] for c in range(0, cols, BLOCK)]
        if case["block_rows"] == 1:
            amax = torch.stack([p.amax(1) for p in parts])
        else:
            amax = torch.stack([torch.stack([p[r:r + BLOCK].amax() for p in parts])
                                for r in range(0, x.shape[0], BLOCK)])
        scale = torch.exp2(torch.floor(torch.log2(amax / 448)) - 1)
        for _ in range(3):
            scale = torch.where(amax / scale > 448, scale * 2, scale)
        return None, torch.where(amax == 0, torch.ones_like(scale), scale.clamp(min=2.0 ** -126))
    column = lambda n: torch.arange(n, device="cuda") // BLOCK  # noqa: E731
    if op in ("linear_fp8", "linear_fp8_grad"):
        n, k = case["n"], case["k"]
        x = s["x8"].to(wide) * s["xs"].to(wide)[column(s["x8"].shape[1])].t()
        w = s["w8"].to(wide) * s["ws"].to(wide)[column(n)][:, column(k)]
        if op == "linear_fp8_grad":
            return torch.matmul(x, w)
        y = torch.matmul(x, w.t())
        return _exact_act(y if s["bias"] is None else y + s["bias"].to(wide), case["act"])
    if op in ("grouped", "grouped_grad"):
        n, k = case["n"], case["k"]
        y = torch.zeros(case["rows"], n if op == "grouped" else k, dtype=wide, device="cuda")
        dw = torch.zeros(case["groups"], n, k, dtype=wide, device="cuda") if op == "grouped_grad" else None
        at = 0
        for g, size in enumerate(s["sizes"]):
            rows = slice(at, at + size)
            w = s["w"][g].to(wide)
            if op == "grouped":
                y[rows] = s["x"][rows].to(wide) @ w.t()
            else:
                dy = s["dy"][rows].to(wide)
                y[rows] = dy @ w
                dw[g] = dy.t() @ s["x"][rows].to(wide)
            at += size
        return y if op == "grouped" else (y, dw)
    x = s["x8"].to(wide) * s["xs"].to(wide)[column(case["k"])].t()
    z = s["z8"].to(wide) * s["zs"].to(wide)[column(case["n"])].t()
    z.requires_grad_(True)
    slope, = torch.autograd.grad(_exact_act(z, case["act"]).sum(), z)
    dz = s["dy"].to(wide) * slope
    return dz @ s["w"].to(wide), dz.t() @ x, dz.sum(0)


def _exact_act(z, name):
    if name == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if name == "gelu":   # 0.5 (1 + tanh u) = sigmoid(2 u)
        return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "sigmoid":
        return torch.sigmoid(z)
    return z * 1.0
