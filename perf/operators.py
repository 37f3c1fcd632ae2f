"""The microscaled 4-bit operators, as a user's program calls them, next to their plain form.

A matrix in this format is quantised along its rows in blocks of 32 consecutive elements (the last block of a row may
be shorter).  A block shares one power-of-two scale 2^e, and each element is a 4-bit e2m1 number (sign and one of
0, 0.5, 1, 1.5, 2, 3, 4, 6):

    e     = floor(log2(max |x|)) - 2, clamped to [-127, 127]   (-127 for a block of zeros)
    value = 2^e * e2m1(x / 2^e)                                (nearest, ties to even, at most 6 in magnitude)

A block that holds an infinity or a NaN becomes NaN as a whole.  What a call keeps in memory:

    codes   uint8 [rows][16 * ceil(cols / 32)]   element 2i in the low half of byte i, zeros past the last column
    scales  uint8, e + 127 (255: NaN); byte ((r / 128) * ceil(blocks / 4) + b / 4) * 512
                                            + (r % 32) * 16 + (r / 32 % 4) * 4 + b % 4   for row r, block b; zeros elsewhere

The operators: quantisation (along the rows, along the columns, or both from one reading), the values back, the
product A . B^T of two quantised matrices, and the same product quantised again by its output stage.
"""
import math

import torch

own = False

DEVICE = "cuda" if torch.cuda.is_available() else "cpu"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}
LARGEST = 8192


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # one new token's activations, before its products: the smallest call
        {"name": "values, one token", "op": "values", "rows": 1, "cols": 4096, "type": "bf16", "way": "rows", "pad": 0},
        # a weight matrix at the start of a training step: forward and backward copies from one reading
        {"name": "values, weights both ways", "op": "values", "rows": 4096, "cols": 4096, "type": "bf16", "way": "both", "pad": 0},
        # a slice of a wider buffer, sizes that no block and no vector divides, blocks along the columns
        {"name": "values, ragged columns", "op": "values", "rows": 1000, "cols": 2999, "type": "f32", "way": "columns", "pad": 13},
        # one token against a kept weight matrix: the bytes of the weights count
        {"name": "product, one token", "op": "product", "m": 1, "n": 4096, "k": 4096, "type": "bf16", "add": False},
        # odd sizes added into a 32-bit buffer, as gradients are summed over pieces of a batch
        {"name": "product, ragged and added", "op": "product", "m": 67, "n": 1001, "k": 4103, "type": "f32", "add": True},
        # a batch of sequences being answered, some hundred tokens a step
        {"name": "product, 512 tokens", "op": "product", "m": 512, "n": 4096, "k": 4096, "type": "bf16", "add": False},
        # the largest product
        {"name": "product, 8192 cubed", "op": "product", "m": 8192, "n": 8192, "k": 8192, "type": "bf16", "add": False},
        # a low-rank or latent projection that feeds the next product in 4 bits: few tokens, and a whole prompt
        {"name": "requantised, 16 tokens", "op": "requantised", "m": 16, "n": 4096, "k": 4096},
        {"name": "requantised, 4096 cubed", "op": "requantised", "m": 4096, "n": 4096, "k": 4096},
        # a layer that serves: activations quantised in the call, weights kept quantised
        {"name": "layer, 64 tokens", "op": "layer", "m": 64, "n": 16384, "k": 4096, "type": "f16"},
        # a training step of one layer: quantise both ways, forward, both gradients
        {"name": "step, 4096 tokens", "op": "step", "m": 4096, "n": 4096, "k": 4096, "type": "bf16"},
        {"name": "step, ragged", "op": "step", "m": 130, "n": 200, "k": 328, "type": "f32"},
    ]


def draw(rng):
    size = lambda least, most=LARGEST: int(round(math.exp(rng.uniform(math.log(least), math.log(most)))))  # noqa: E731
    op = rng.choice(["values", "product", "requantised", "layer", "step"])
    kind = rng.choice(sorted(TYPES))
    if op == "values":
        return {"op": op, "rows": size(1), "cols": size(8), "type": kind, "way": rng.choice(["rows", "columns", "both"]),
                "pad": rng.choice([0, 0, 8, 13])}
    case = {"op": op, "m": size(1), "n": size(8), "k": size(8)}
    if op == "product":
        case.update(type=kind, add=kind == "f32" and rng.random() < 0.5)
    elif op == "layer":
        case.update(type=kind)
    elif op == "step":
        case.update(m=size(1, 4096), n=size(8, 4096), k=size(8, 4096), type=kind)
    return case


def work(case):
    held = lambda rows, cols: rows * cols * 17 / 32  # noqa: E731  codes and scales
    if case["op"] == "values":
        n = case["rows"] * case["cols"]
        out = BYTES[case["type"]] if case["type"] == "f32" else 2
        return {"bytes": n * BYTES[case["type"]] + n * out * (2 if case["way"] == "both" else 1), "flops": n}
    m, n, k = case["m"], case["n"], case["k"]
    if case["op"] == "product":
        return {"bytes": held(m, k) + held(n, k) + m * n * BYTES[case["type"]] * (2 if case["add"] else 1), "flops": 2 * m * n * k}
    if case["op"] == "requantised":
        return {"bytes": held(m, k) + held(n, k) + 2 * m * n, "flops": 2 * m * n * k}
    b = BYTES[case["type"]]
    if case["op"] == "layer":
        return {"bytes": m * k * b + held(n, k) + m * n * b, "flops": 2 * m * n * k}
    return {"bytes": b * 2 * (m * k + m * n) + b * n * k + 4 * n * k, "flops": 6 * m * n * k}


# ------------------------------------------------------------------------------------------------ the inputs
def _activations(rows, cols, g):
    """Normal values times a spread of the columns, a few columns far larger, and a row of zeros (padding)."""
    spread = torch.exp(0.4 * torch.randn(cols, generator=g, device=DEVICE))
    spread = torch.where(torch.rand(cols, generator=g, device=DEVICE) < 0.004, 8 * spread, spread)
    x = torch.randn(rows, cols, generator=g, device=DEVICE) * spread
    if rows > 4:
        x[rows // 2] = 0
    return x


def _weights(rows, cols, g):
    return 0.02 * torch.randn(rows, cols, generator=g, device=DEVICE)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(int(seed))
    s = dict(case)
    if case["op"] == "values":
        wide = _activations(case["rows"], case["cols"] + case["pad"], g).to(TYPES[case["type"]])
        s["x"] = wide[:, :case["cols"]]
        return s
    m, n, k = case["m"], case["n"], case["k"]
    if case["op"] in ("product", "requantised"):
        s["a"] = _pack(_activations(m, k, g))
        s["b"] = _pack(_weights(n, k, g))
        if case["op"] == "product" and case["add"]:
            s["c"] = torch.randn(m, n, generator=g, device=DEVICE)
    elif case["op"] == "layer":
        s["x"] = _activations(m, k, g).to(TYPES[case["type"]])
        s["w"] = _pack(_weights(n, k, g))
    else:
        s["x"] = _activations(m, k, g).to(TYPES[case["type"]])
        s["w"] = _weights(n, k, g).to(TYPES[case["type"]])
        s["dy"] = (0.001 * _activations(m, n, g)).to(TYPES[case["type"]])
    return s


# ------------------------------------------------------------------------------------------------ the plain forms
def _power(e):
    """2^e in 32 bits for whole e in [-127, 127]."""
    return torch.where(e > -127, (e + 127) << 23, torch.full_like(e, 1 << 22)).view(torch.float32)


def _split(x):
    """x in 32 bits [rows][cols] as whole exponents [rows][blocks] (128: the block is NaN) and magnitudes, with signs,
    on the e2m1 grid [rows][blocks][32]."""
    rows, cols = x.shape
    blocks = -(-cols // 32)
    full = torch.zeros(rows, blocks * 32, dtype=torch.float32, device=x.device)
    full[:, :cols] = x
    full = full.view(rows, blocks, 32)
    most = full.abs().amax(-1)
    bad = ~torch.isfinite(full).all(-1)
    most = torch.where(bad, torch.zeros_like(most), most)
    e = torch.where(most > 0, torch.frexp(most)[1] - 3, torch.full_like(most, -127, dtype=torch.int32)).clamp(-127, 127)
    y = torch.where(bad[..., None], torch.zeros_like(full), full) * _power(-e)[..., None]
    step = torch.where(y.abs() < 2, 0.5, torch.where(y.abs() < 4, 1.0, 2.0))
    q = (torch.round(y / step) * step).clamp(-6, 6)
    return torch.where(bad, torch.full_like(e, 128), e), q


def _values(x):
    e, q = _split(x.float())
    v = q * torch.where(e == 128, torch.full_like(q[..., 0], float("nan")), _power(e.clamp(max=127)))[..., None]
    return v.reshape(x.shape[0], -1)[:, :x.shape[1]]


def _pack(x):
    """A quantised matrix as it is kept: codes and scales."""
    e, q = _split(x)
    rows, blocks = e.shape
    a = q.abs()
    code = torch.where(a <= 2, 2 * a, torch.where(a == 3, 5.0, torch.where(a == 4, 6.0, 7.0))).to(torch.uint8)
    code = (code | (torch.signbit(q).to(torch.uint8) << 3)).view(rows, blocks * 16, 2)
    high, wide = -(-rows // 128), -(-blocks // 4)
    s = torch.zeros(high * 128, wide * 4, dtype=torch.uint8, device=x.device)
    s[:rows, :blocks] = (e + 127).to(torch.uint8)
    s = s.view(high, 4, 32, wide, 4).permute(0, 3, 2, 1, 4).contiguous().view(-1)
    return {"codes": code[..., 0] | (code[..., 1] << 4), "scales": s, "rows": rows, "cols": x.shape[1]}


def _unpack(p):
    rows, cols = p["rows"], p["cols"]
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], device=DEVICE)
    codes = p["codes"].int()
    v = grid[torch.stack([codes & 15, codes >> 4], -1)].view(rows, -1, 32)
    wide = -(-v.shape[1] // 4)
    s = p["scales"].view(-1, wide, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(-1, wide * 4)[:rows, :v.shape[1]].int()
    scale = torch.where(s == 255, torch.full_like(v[..., 0], float("nan")), _power(s.clamp(max=254) - 127))
    return (v * scale[..., None]).view(rows, -1)[:, :cols]


def _value_type(case):
    return torch.float32 if case["type"] == "f32" else torch.bfloat16


def run(s):
    if own:
        return _run_own(s)
    if s["op"] == "values":
        out = {}
        if s["way"] != "columns":
            out["rows"] = _values(s["x"]).to(_value_type(s))
        if s["way"] != "rows":
            out["columns"] = _values(s["x"].t()).to(_value_type(s))
        return out
    if s["op"] == "product":
        c = _unpack(s["a"]) @ _unpack(s["b"]).t()
        if s["add"]:
            s["c"] += c
            return s["c"]
        return c.to(TYPES[s["type"]])
    if s["op"] == "requantised":
        return _values(_unpack(s["a"]) @ _unpack(s["b"]).t()).to(torch.bfloat16)
    t = TYPES[s["type"]]
    if s["op"] == "layer":
        return (_values(s["x"]) @ _unpack(s["w"]).t()).to(t)
    x, w, dy = s["x"], s["w"], s["dy"]
    return {"y": (_values(x) @ _values(w).t()).to(t),
            "dx": (_values(dy) @ _values(w.t()).t()).to(t),
            "dw": _values(dy.t()) @ _values(x.t()).t()}


# ------------------------------------------------------------------------------------------------ the framework's calls
_contexts = []


def _run_own(s):
    from aiehlc_b200.ops import Context, MxFp4
    if not _contexts:
        _contexts.append(Context(0))
    ctx = _contexts[0]
    held = lambda p: MxFp4(p["codes"], p["scales"], p["rows"], p["cols"])  # noqa: E731
    if s["op"] == "values":
        t = _value_type(s)
        if s["way"] == "rows":
            return {"rows": ctx.dequantize_mxfp4(ctx.quantize_mxfp4(s["x"]), t)}
        if s["way"] == "columns":
            return {"columns": ctx.dequantize_mxfp4(ctx.quantize_mxfp4(s["x"], "columns"), t)}
        r, c = ctx.quantize_mxfp4(s["x"], "both")
        return {"rows": ctx.dequantize_mxfp4(r, t), "columns": ctx.dequantize_mxfp4(c, t)}
    if s["op"] == "product":
        if s["add"]:
            return ctx.gemm_mxfp4(held(s["a"]), held(s["b"]), out=s["c"], accumulate=True)
        return ctx.gemm_mxfp4(held(s["a"]), held(s["b"]), TYPES[s["type"]])
    if s["op"] == "requantised":
        return ctx.dequantize_mxfp4(ctx.gemm_mxfp4_mxfp4(held(s["a"]), held(s["b"])), torch.bfloat16)
    t = TYPES[s["type"]]
    if s["op"] == "layer":
        return ctx.gemm_mxfp4(ctx.quantize_mxfp4(s["x"]), held(s["w"]), t)
    x, xt = ctx.quantize_mxfp4(s["x"], "both")
    w, wt = ctx.quantize_mxfp4(s["w"], "both")
    y = ctx.gemm_mxfp4(x, w, t)
    dy, dyt = ctx.quantize_mxfp4(s["dy"], "both")
    return {"y": y, "dx": ctx.gemm_mxfp4(dy, wt, t), "dw": ctx.gemm_mxfp4(dyt, xt, torch.float32)}


# ------------------------------------------------------------------------------------------------ 64 bits
def _two_to(e):
    """2^e in 64 bits, built from its bits (a device's pow() may be one step off)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_values(x):
    """The definition, in 64 bits: the block's exponent by comparisons of powers of two, each element's code by counting
    the borders below it (a border itself belongs to the even code beside it)."""
    x = x.double()
    rows, cols = x.shape
    x = torch.nn.functional.pad(x, (0, -cols % 32)).reshape(rows, -1, 32)
    fine = torch.isfinite(x).all(dim=2, keepdim=True)
    x = torch.nan_to_num(x, 0.0, 0.0, 0.0) * fine
    most = x.abs().max(dim=2, keepdim=True).values
    e = torch.floor(torch.log2(most.clamp(min=2.0 ** -1000)))
    e = e - (_two_to(e) > most).double()
    e = e + (_two_to(e + 1) <= most).double()
    scale = _two_to((e - 2).clamp(-127, 127))
    y = x.abs() / scale
    table = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    v = torch.zeros_like(y)
    for i in range(7):
        border = (table[i] + table[i + 1]) / 2
        v = v + (table[i + 1] - table[i]) * ((y >= border) if i % 2 else (y > border)).double()
    v = torch.where(fine, torch.copysign(v, x) * scale, torch.full_like(v, float("nan")))
    return v.reshape(rows, -1)[:, :cols]


def _exact_unpack(p):
    rows, cols = p["rows"], p["cols"]
    j = torch.arange(cols, device=DEVICE)
    r = torch.arange(rows, device=DEVICE)[:, None]
    code = (p["codes"].long()[:, j // 2] >> (4 * (j % 2))) & 15
    high, low = (code >> 1) & 3, code & 1
    v = torch.where(high == 0, 0.5 * low.double(), (1 + 0.5 * low.double()) * _two_to(high - 1))
    v = torch.where(code > 7, -v, v)
    blocks = -(-cols // 32)
    b = torch.arange(blocks, device=DEVICE)
    at = ((r // 128) * (-(-blocks // 4)) + b // 4) * 512 + (r % 32) * 16 + (r // 32 % 4) * 4 + b % 4
    s = p["scales"].long()[at]
    scale = torch.where(s == 255, float("nan"), _two_to(s - 127))
    return v * scale[:, j // 32]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "values":
        out = {}
        if case["way"] in ("rows", "both"):
            out["rows"] = _exact_values(s["x"])
        if case["way"] in ("columns", "both"):
            out["columns"] = _exact_values(s["x"].t())
        return out
    if case["op"] == "product":
        c = torch.matmul(_exact_unpack(s["a"]), _exact_unpack(s["b"]).t())
        return c + s["c"].double() if case["add"] else c
    if case["op"] == "requantised":
        return _exact_values(torch.matmul(_exact_unpack(s["a"]), _exact_unpack(s["b"]).t()))
    if case["op"] == "layer":
        return torch.matmul(_exact_values(s["x"]), _exact_unpack(s["w"]).t())
    return {"y": torch.matmul(_exact_values(s["x"]), _exact_values(s["w"]).t()),
            "dx": torch.matmul(_exact_values(s["dy"]), _exact_values(s["w"].t()).t()),
            "dw": torch.matmul(_exact_values(s["dy"].t()), _exact_values(s["x"].t()).t())}
