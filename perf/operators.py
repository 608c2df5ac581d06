"""Timed cases of the microscaled operators (``ancha_amd.mx``): values in blocks of 32 along the
reduction axis that share a power of two, held as e4m3 ("fp8") or e2m1 ("fp4") codes.

  norm      mx.unit_norm / mx.add_unit_norm   row norm, with the residual's addition, to 8 (or 4) bits
  quantize  mx.quantize / mx.weight           activations along their rows, a weight along its k axis
  linear    mx.linear                         8- or 4-bit rows . 4-bit weight with its epilogue

``run`` is one pass: the elementary form in torch where ``own`` is false, the framework's calls where
it is true. Codes come back as the values they stand for (``values()``).
"""
import math

import torch

own = False

DEVICE = "cuda"
BLOCK = 32
TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
WIDTH = {"float32": 4, "float16": 2, "bfloat16": 2, "fp8": 1 + 1 / 32, "fp4": 0.5 + 1 / 32}
# Per format: exponent of the largest value, exponent of the smallest normal one, mantissa bits, largest value.
FORMATS = {"fp8": (8, -6, 3, 448.0), "fp4": (2, 0, 1, 6.0)}
HEAD = 64


def listed():
    return [
        # One token of a served model between two layers.
        {"name": "norm_token", "op": "norm", "rows": 1, "dim": 4096, "type": "bfloat16", "add": True,
         "eps": 1e-6, "format": "fp8"},
        # The norm between layers over two 8 s chunks of the bundled Mel model (120 x 801 rows).
        {"name": "norm_layers", "op": "norm", "rows": 96120, "dim": 384, "type": "float32", "add": True,
         "eps": 0.0, "format": "fp8"},
        # One chunk's rows at an odd width, straight to 4 bits.
        {"name": "norm_odd", "op": "norm", "rows": 6007, "dim": 1549, "type": "float16", "add": False,
         "eps": 1e-5, "format": "fp4"},
        # The activations of a few tokens: launch and latency.
        {"name": "quantize_tokens", "op": "quantize", "kind": "rows", "rows": 4, "dim": 512,
         "type": "float32", "format": "fp8"},
        # A long prompt's wide activations.
        {"name": "quantize_prompt", "op": "quantize", "kind": "rows", "rows": 16384, "dim": 8192,
         "type": "bfloat16", "format": "fp4"},
        # A wide projection's weight, once at load time ([out, in] storage seen as [in, out]).
        {"name": "quantize_weight", "op": "quantize", "kind": "weight", "rows": 8192, "dim": 8192,
         "type": "float32", "format": "fp4"},
        # One token through a projection.
        {"name": "linear_token", "op": "linear", "n": 1, "k": 4096, "m": 4096, "format": "fp8",
         "out": "bfloat16", "bias": True, "gelu": False, "rotary": 0, "residual": True},
        # A batch of tokens served together: the weight is what has to be read.
        {"name": "linear_batch", "op": "linear", "n": 24, "k": 8192, "m": 8192, "format": "fp4",
         "out": "bfloat16", "bias": False, "gelu": False, "rotary": 0, "residual": False},
        # Odd sizes on every axis.
        {"name": "linear_odd", "op": "linear", "n": 801, "k": 1000, "m": 1549, "format": "fp8",
         "out": "float16", "bias": True, "gelu": False, "rotary": 0, "residual": False},
        # The feed-forward's first projection over two 8 s chunks, its hidden rows kept in 8 bits.
        {"name": "linear_ff_in", "op": "linear", "n": 96120, "k": 384, "m": 1536, "format": "fp8",
         "out": "fp8", "bias": True, "gelu": True, "rotary": 0, "residual": False},
        # The feed-forward's second projection over two 8 s chunks, onto the residual stream.
        {"name": "linear_ff_out", "op": "linear", "n": 96120, "k": 1536, "m": 384, "format": "fp8",
         "out": "float32", "bias": True, "gelu": False, "rotary": 0, "residual": True},
        # A long prompt through a wide projection: bound by the matrix cores.
        {"name": "linear_prompt", "op": "linear", "n": 8192, "k": 8192, "m": 8192, "format": "fp8",
         "out": "bfloat16", "bias": False, "gelu": False, "rotary": 0, "residual": False},
    ]


def _spread(rng, low, high):
    """A whole number in low..high, spread over the logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("norm", "quantize", "linear"))
    if op == "norm":
        dim = _spread(rng, 64, 16384)
        return {"op": op, "rows": _spread(rng, 1, min(100_000, (1 << 27) // dim)), "dim": dim,
                "type": rng.choice(list(TYPES)), "add": rng.random() < 0.7,
                "eps": rng.choice((0.0, 1e-6, 1e-5)), "format": rng.choice(("fp8", "fp8", "fp4"))}
    if op == "quantize":
        kind = rng.choice(("rows", "rows", "weight"))
        dim = _spread(rng, 32, 16384)
        most = min(16384, (1 << 26) // dim) if kind == "weight" else min(100_000, (1 << 27) // dim)
        return {"op": op, "kind": kind, "rows": _spread(rng, 16 if kind == "weight" else 1, most),
                "dim": dim, "type": rng.choice(list(TYPES)),
                "format": "fp4" if kind == "weight" else rng.choice(("fp8", "fp4"))}
    k, m = _spread(rng, 64, 8192), _spread(rng, 64, 8192)
    n = _spread(rng, 1, min(100_000, (1 << 39) // (k * m)))
    out = rng.choice(("float32", "float16", "bfloat16", "fp8"))
    rotary = 0
    if rng.random() < 0.2 and out != "fp8":
        # The q | k | v projection of some heads, rotated at its end.
        heads = max(1, min(m // (3 * HEAD), 16))
        rotary, m = HEAD * heads, max(m, 3 * HEAD * heads)
    return {"op": op, "n": n, "k": k, "m": m, "format": rng.choice(("fp8", "fp4")), "out": out,
            "bias": rng.random() < 0.6, "gelu": rotary == 0 and rng.random() < 0.3, "rotary": rotary,
            "residual": rotary == 0 and rng.random() < 0.4}


def work(case):
    """Bytes and operations that a pass cannot do without: inputs read once, outputs written once."""
    if case["op"] == "linear":
        n, k, m = case["n"], case["k"], case["m"]
        out = 2 if case["out"] == "fp8" else WIDTH[case["out"]]
        byt = n * k * WIDTH[case["format"]] + k * m * WIDTH["fp4"] + n * m * out
        if case["bias"]:
            byt += 4 * m
        if case["rotary"]:
            byt += 4 * 4 * HEAD * _tokens(n)
        if case["residual"]:
            byt += n * m * (4 if case["out"] == "fp8" else WIDTH[case["out"]])
        return {"bytes": byt, "flops": 2 * n * k * m}
    values = case["rows"] * case["dim"]
    width = WIDTH[case["type"]]
    if case["op"] == "quantize":  # the values come back in 16 bits
        return {"bytes": values * (width + 2), "flops": 4 * values}
    adds = 2 * width if case["add"] else 0  # the residual read, the sum written
    return {"bytes": values * (width + adds + 2) + 4 * case["dim"], "flops": 8 * values}


def _tokens(n):
    """Rotary positions of n rows: the largest divisor of n up to 2048."""
    return max(t for t in range(1, min(n, 2048) + 1) if n % t == 0)


def _table(tokens):
    """The packed rotary table [4, tokens, 64]: query cosine and signed sine (both / 8), the key's."""
    freqs = 10000.0 ** (-torch.arange(HEAD // 2, dtype=torch.float64, device=DEVICE) / (HEAD // 2))
    angle = torch.arange(tokens, dtype=torch.float64, device=DEVICE)[:, None] * freqs
    cos = angle.cos().repeat_interleave(2, 1)
    sin = torch.stack((-angle.sin(), angle.sin()), 2).reshape(tokens, HEAD)
    return torch.stack((cos / 8, sin / 8, cos, sin)).float().contiguous()


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device=DEVICE)

    s = {"case": case}
    if case["op"] == "linear":
        n, k, m = case["n"], case["k"], case["m"]
        # Activations as a norm leaves them, with some channels larger than the rest.
        x = normal(n, k) * (1 + 4 * (normal(k).abs() > 2))
        w = normal(m, k) / math.sqrt(k)
        s["x"], s["w"] = _encode(x, case["format"]), _encode(w, "fp4")
        s["k"] = k
        if case["bias"]:
            s["bias"] = 0.1 * normal(m)
        if case["rotary"]:
            s["table"] = _table(_tokens(n))
        if case["residual"]:
            s["residual"] = normal(n, m).to(TYPES.get(case["out"], torch.float32))
        if own:
            from ancha_amd import mx
            s["x"] = mx.Tensor(*s["x"], case["format"], (n, k))
            s["w"] = mx.weight(w.t())
        return s
    rows, dim = case["rows"], case["dim"]
    dtype = TYPES[case["type"]]
    if case["op"] == "quantize" and case["kind"] == "weight":
        s["x"] = (normal(dim, rows) / math.sqrt(rows)).to(dtype).t()  # [in, out] view of [out, in]
        return s
    s["x"] = (normal(rows, dim) * (1 + 4 * (normal(dim).abs() > 2))).to(dtype)
    if case["op"] == "norm":
        s["scale"] = math.sqrt(dim) * (1 + 0.2 * normal(dim))
        if case["add"]:
            s["residual"] = (normal(rows, dim) * 2).to(dtype)
    return s


# The plain form.


def _pad(dim):
    """Columns of a row as it is stored: whole groups of four blocks, zeros behind the last value."""
    return -(-dim // (4 * BLOCK)) * 4 * BLOCK


def _round(x, fmt):
    """x [rows, dim], 32 or 64 bits -> (rounded values in units of the scale, scale codes) per block."""
    top, low, bits, most = FORMATS[fmt]
    rows, dim = x.shape
    blocks = torch.nn.functional.pad(x, (0, _pad(dim) - dim)).reshape(rows, -1, BLOCK)
    largest = blocks.abs().amax(2, keepdim=True)
    exponent = torch.frexp(largest).exponent - 1  # floor(log2)
    scale = torch.where(largest > 0, (exponent - top).clamp(min=-127), -127)
    v = torch.ldexp(blocks, -scale)
    step = torch.frexp(v).exponent - 1
    step = torch.where(v != 0, step, low).clamp(min=low) - bits
    q = torch.ldexp(torch.ldexp(v, -step).round(), step).clamp(-most, most)
    return q, scale


def _encode(x, fmt):
    """(codes, scales) of x [rows, dim] as a program holds them: one byte per e4m3 value, two e2m1
    values to a byte (the first in its low half), one byte 127 + exponent per block."""
    q, scale = _round(x, fmt)
    rows = x.shape[0]
    scales = (scale + 127).to(torch.uint8).reshape(rows, -1)
    q = q.reshape(rows, -1)
    if fmt == "fp8":
        return q.to(torch.float8_e4m3fn).view(torch.uint8), scales
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=x.device)
    code = torch.searchsorted(grid, q.abs().contiguous()) + 8 * torch.signbit(q)
    return (code[:, 0::2] + 16 * code[:, 1::2]).to(torch.uint8), scales


def _decode(codes, scales, fmt, dim):
    """The 32-bit values [rows, dim] that codes and scales stand for."""
    rows = codes.shape[0]
    if fmt == "fp8":
        v = codes.view(torch.float8_e4m3fn).float()
    else:
        grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
        both = torch.stack((codes & 15, codes >> 4), 2).reshape(rows, -1).long()
        v = grid[both & 7] * (1 - 2 * (both >> 3))
    v = torch.ldexp(v.reshape(rows, -1, BLOCK), scales.int()[:, :, None] - 127)
    return v.reshape(rows, -1)[:, :dim]


def _values(x, fmt):
    """The values [rows, dim] after rounding to the format; 16 bits hold them exactly."""
    q, scale = _round(x, fmt)
    return torch.ldexp(q, scale).reshape(x.shape[0], -1)[:, :x.shape[1]].to(torch.bfloat16)


def _rotate(y, table, width):
    """Query columns [0, width) and key columns [width, 2 width) of rows at position r % tokens."""
    tokens = table.shape[1]
    at = torch.arange(y.shape[0], device=y.device) % tokens
    out = [y[:, 2 * width:]]
    for part in (1, 0):
        x = y[:, part * width:(part + 1) * width].reshape(y.shape[0], -1, HEAD)
        cos, sin = table[2 * part][at][:, None], table[2 * part + 1][at][:, None]
        swapped = torch.stack((x[..., 1::2], x[..., 0::2]), 3).reshape(x.shape)
        out.insert(0, (x * cos + swapped * sin).reshape(y.shape[0], width))
    return torch.cat(out, 1)


def _linear_plain(s):
    case = s["case"]
    y = _decode(*s["x"], case["format"], s["k"]) @ _decode(*s["w"], "fp4", s["k"]).t()
    if case["bias"]:
        y = y + s["bias"]
    if case["gelu"]:
        y = 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    if case["rotary"]:
        y = _rotate(y, s["table"], case["rotary"])
    if case["residual"]:
        y = y + s["residual"].float()
    return _values(y, "fp8") if case["out"] == "fp8" else y.to(TYPES[case["out"]])


def _plain(s):
    case, x = s["case"], s.get("x")
    if case["op"] == "linear":
        return _linear_plain(s)
    if case["op"] == "quantize":
        if case["kind"] == "weight":
            return _values(x.t().float(), "fp4").t()
        return _values(x.float(), case["format"])
    total = (x.float() + s["residual"].float()).to(x.dtype) if case["add"] else x
    # 64 bits: a rounding to 32 before the one to 8 or 4 would move values next to a border.
    h = total.double()
    length = (h.square().sum(1, keepdim=True) + case["dim"] * case["eps"]).sqrt().clamp(min=1e-12)
    y = _values(h / length * s["scale"].double(), case["format"])
    return (y, total) if case["add"] else y


def _own(s):
    from ancha_amd import fused, mx

    case = s["case"]
    if case["op"] == "linear":
        epilogue = fused.Epilogue(bias=s.get("bias"), gelu=case["gelu"], residual=s.get("residual"),
                                  rotary=(s["table"], case["rotary"]) if case["rotary"] else None)
        if case["out"] == "fp8":
            return mx.linear(s["x"], s["w"], epilogue, format="fp8").values(torch.bfloat16)
        return mx.linear(s["x"], s["w"], epilogue, dtype=TYPES[case["out"]])
    if case["op"] == "quantize":
        if case["kind"] == "weight":
            return mx.weight(s["x"]).values(torch.bfloat16)
        return mx.quantize(s["x"], case["format"]).values(torch.bfloat16)
    if case["add"]:
        y, total = mx.add_unit_norm(s["x"], s["residual"], s["scale"], eps=case["eps"],
                                    format=case["format"])
        return y.values(torch.bfloat16), total
    return mx.unit_norm(s["x"], s["scale"], eps=case["eps"],
                        format=case["format"]).values(torch.bfloat16)


def run(state):
    return _own(state) if own else _plain(state)


# The definition in 64 bits, by the list of the values that a format has.


def _grid(fmt):
    """The format's non-negative values in the order of their codes."""
    top, low, bits, most = FORMATS[fmt]
    values = [m * 2.0 ** (low - bits) for m in range(2 ** bits)]
    values += [(1 + m / 2 ** bits) * 2.0 ** e for e in range(low, top + 1) for m in range(2 ** bits)]
    return torch.tensor([v for v in values if v <= most], dtype=torch.float64, device=DEVICE)


def _nearest(x, fmt):
    """x [rows, dim] in 64 bits -> the nearest values of the format under each block's scale."""
    grid = _grid(fmt)
    border = (grid[1:] + grid[:-1]) / 2
    rows, dim = x.shape
    full = torch.zeros(rows, -(-dim // BLOCK) * BLOCK, dtype=torch.float64, device=x.device)
    full[:, :dim] = x
    full = full.reshape(-1, BLOCK)
    scale = torch.exp2(torch.floor(torch.log2(full.abs().max(1, keepdim=True).values)) - FORMATS[fmt][0])
    # log2 rounds: the power of two has to be the largest that is not above the block's largest value.
    largest = full.abs().max(1, keepdim=True).values / 2.0 ** FORMATS[fmt][0]
    scale = torch.where(scale > largest, scale / 2, torch.where(2 * scale <= largest, 2 * scale, scale))
    scale = scale.clamp(min=2.0 ** -127)
    size = full.abs() / scale
    below, above = torch.bucketize(size, border), torch.bucketize(size, border, right=True)
    code = torch.where(below % 2 == 0, below, above)  # a tie goes to the even code
    return (torch.sign(full) * grid[code] * scale).reshape(rows, -1)[:, :dim]


def _exact_operand(pair, fmt, dim):
    """Stored codes and scales as 64-bit values."""
    codes, scales = pair
    grid = _grid(fmt)
    c = codes.long()
    if fmt == "fp4":
        c = torch.stack((c % 16, c // 16), 2).reshape(c.shape[0], -1)
    half = 8 if fmt == "fp4" else 128
    v = torch.where(c >= half, -grid[(c % half).clamp(max=len(grid) - 1)],
                    grid[(c % half).clamp(max=len(grid) - 1)])
    v *= torch.exp2(scales.double() - 127).repeat_interleave(BLOCK, 1)
    return v[:, :dim]


def exact(case, seed):
    s = _prepare_plain(case, seed)
    if case["op"] == "linear":
        n, m = case["n"], case["m"]
        y = torch.matmul(_exact_operand(s["x"], case["format"], case["k"]),
                         _exact_operand(s["w"], "fp4", case["k"]).t().contiguous())
        if case["bias"]:
            y += s["bias"].double()
        if case["gelu"]:
            y = y * torch.special.ndtr(y)
        if case["rotary"]:
            heads = case["rotary"] // HEAD
            z = y[:, :2 * case["rotary"]].reshape(n, 2, heads, HEAD // 2, 2)
            t = s["table"].double()[:, torch.arange(n, device=DEVICE) % s["table"].shape[1]]
            cos = torch.stack((t[0], t[2]), 1).reshape(n, 2, 1, HEAD // 2, 2)
            sin = torch.stack((t[1], t[3]), 1).reshape(n, 2, 1, HEAD // 2, 2)
            y = torch.cat(((z * cos + z.flip(4) * sin).reshape(n, -1), y[:, 2 * case["rotary"]:]), 1)
        if case["residual"]:
            y = y + s["residual"].double()
        return _nearest(y, "fp8") if case["out"] == "fp8" else y
    x = s["x"].double()
    if case["op"] == "quantize":
        if case["kind"] == "weight":
            return _nearest(x.t().contiguous(), "fp4").t()
        return _nearest(x, case["format"])
    if case["add"]:
        total = (s["x"].float() + s["residual"].float()).to(s["x"].dtype)  # a rounding of its own
        x = total.double()
    y = x / torch.sqrt((x * x).sum(1) + case["dim"] * case["eps"]).clamp(min=1e-12)[:, None]
    y = _nearest(y * s["scale"].double(), case["format"])
    return (y, x) if case["add"] else y


def _prepare_plain(case, seed):
    """prepare()'s inputs as the plain form has them."""
    global own
    before, own = own, False
    try:
        return prepare(case, seed)
    finally:
        own = before
