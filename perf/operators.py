"""Measured cases of the 4-bit floating point linear layer and of the layer norm in front of it.

Four operators, as a program that serves a quantized layer, or tunes adapters around it, calls them:

* ``layer_norm``  affine layer norm; with ``train`` its backward pass too, the weight's and bias's
  gradients reduced over all rows;
* ``quantize``    rows to 4-bit floating point with a scale per block, after the 256-wide ConvRot
  rotation or without it, and the values read back;
* ``linear``      the product of two quantized operands, bias added, from one token to long sequences;
* ``grad_input``  the gradient that the layer passes down through its frozen 4-bit weights.

Formats.  ``nvfp4``: blocks of 16 e2m1 codes, an e4m3 scale each, and a power-of-two fp32 scale per
row.  ``mxfp4``: blocks of 32 e2m1 codes, an e8m0 (power of two) scale each; the row scale is 1.
Two codes share a byte, the even column in the low nibble.  Block scales lie in tiles of 128 rows by
four blocks: ``[rows / 128, blocks / 4, 32, 16]``, where row ``32 j + l`` and block ``b`` of a tile sit
at ``[l, 4 j + b]``; what a tile has beyond the tensor is zero bytes.
"""

import math
import sys

import torch

own = False

if "comfyui-turing-utils_b200" not in sys.path:
    sys.path.insert(0, "comfyui-turing-utils_b200")

BLOCK = {"nvfp4": 16, "mxfp4": 32}
SCALE_TYPE = {"nvfp4": torch.float8_e4m3fn, "mxfp4": torch.float8_e8m0fnu}
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPSILON = 1.0e-5


# ---------------------------------------------------------------------------------------- cases
def listed():
    return [
        # A whole 32760-token video sequence through a block's affine norm, inference.
        {"name": "ln_long", "op": "layer_norm", "rows": 32760, "hidden": 5120, "type": "bf16", "weight": "bf16", "train": False},
        # One training step of the same norm on a shard of 4096 tokens, fp32 master weights.
        {"name": "ln_train", "op": "layer_norm", "rows": 4096, "hidden": 5120, "type": "bf16", "weight": "fp32", "train": True},
        # Odd rows and width in full precision: no vector load lines up with a row.
        {"name": "ln_train_odd", "op": "layer_norm", "rows": 2047, "hidden": 1537, "type": "fp32", "weight": "fp32", "train": True},
        # The activations of a long sequence before an attention projection.
        {"name": "quant_long", "op": "quantize", "rows": 32760, "k": 5120, "type": "bf16", "format": "nvfp4", "rotation": 256},
        # The FFN's wide rows, an odd number of them, fp16, without rotation.
        {"name": "quant_wide", "op": "quantize", "rows": 4097, "k": 13824, "type": "fp16", "format": "mxfp4", "rotation": 0},
        # One token on its way to a projection: latency.
        {"name": "quant_token", "op": "quantize", "rows": 1, "k": 5120, "type": "bf16", "format": "nvfp4", "rotation": 256},
        # One token through a projection: the weights are streamed once.
        {"name": "linear_token", "op": "linear", "m": 1, "n": 5120, "k": 5120, "format": "nvfp4", "bias": True},
        # A small batch of tokens into the FFN, the other format.
        {"name": "linear_tokens", "op": "linear", "m": 17, "n": 13824, "k": 5120, "format": "mxfp4", "bias": False},
        # A short prompt with sizes that end inside every tile.
        {"name": "linear_prompt", "op": "linear", "m": 1025, "n": 1537, "k": 1568, "format": "nvfp4", "bias": True},
        # The long sequence into the FFN, the largest product.
        {"name": "linear_long", "op": "linear", "m": 32760, "n": 13824, "k": 5120, "format": "nvfp4", "bias": True},
        # Gradients of a training shard through the rotated attention projection.
        {"name": "grad_proj", "op": "grad_input", "m": 4096, "n": 5120, "k": 5120, "format": "nvfp4", "rotation": 256},
        # A few hundred tokens' gradients through an unrotated FFN weight.
        {"name": "grad_ffn", "op": "grad_input", "m": 333, "n": 13824, "k": 5120, "format": "mxfp4", "rotation": 0},
    ]


def _spread(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["layer_norm", "quantize", "linear", "linear", "grad_input"])
    fmt = rng.choice(["nvfp4", "mxfp4"])
    if op == "layer_norm":
        hidden = _spread(rng, 64, 13824)
        rows = _spread(rng, 1, min(32760, 32760 * 5120 // hidden))
        kind = rng.choice(["bf16", "fp16", "fp32"])
        train = rng.random() < 0.6 and rows * hidden <= 16384 * 5120
        return {"op": op, "rows": rows, "hidden": hidden, "type": kind, "weight": rng.choice([kind, "fp32"]), "train": train}
    rotation = rng.choice([0, 256])
    step = rotation or 32
    k = max(1, _spread(rng, 256, 13824) // step) * step
    if op == "quantize":
        rows = _spread(rng, 1, min(32760, 32760 * 5120 // k))
        return {"op": op, "rows": rows, "k": k, "type": rng.choice(["bf16", "fp16"]), "format": fmt, "rotation": rotation}
    if op == "linear":
        n = _spread(rng, 64, 13824)
        m = _spread(rng, 1, min(32760, 32760 * 13824 * 5120 // (n * k)))
        return {"op": op, "m": m, "n": n, "k": k, "format": fmt, "bias": rng.random() < 0.5}
    n = _spread(rng, 64, 13824) // 8 * 8
    m = _spread(rng, 1, min(16384, 8192 * 13824 * 5120 // (n * k)))
    return {"op": op, "m": m, "n": n, "k": k, "format": fmt, "rotation": rotation}


# ---------------------------------------------------------------------------------------- formats
def _tiles(scales):
    """Plain ``[rows, blocks]`` bytes to tiles of 128 rows by four blocks."""
    rows, blocks = scales.shape
    mt, kt = -(-rows // 128), -(-blocks // 4)
    full = scales.new_zeros((mt * 128, kt * 4))
    full[:rows, :blocks] = scales
    return full.view(mt, 4, 32, kt, 4).permute(0, 3, 2, 1, 4).reshape(mt, kt, 32, 16)


def _untile(tiles, rows, blocks):
    mt, kt = tiles.shape[:2]
    flat = tiles.view(torch.uint8).view(mt, kt, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(mt * 128, kt * 4)
    return flat[:rows, :blocks]


def _rotate(x):
    """The 256-wide rotation of fp32 rows: four radix-4 stages at strides 1, 4, 16 and 64, the four
    halvings taken first (they are exact).  Sums keep this order: the codes hang on their last bit."""
    y = (x * 0.0625).view(-1, 4, 4, 4, 4)
    for dim in (4, 3, 2, 1):
        x0, x1, x2, x3 = y.unbind(dim)
        t, b = x0 + x1, x0 - x1
        y = torch.stack(((t + x2) - x3, (t - x2) + x3, (b + x2) + x3, (x2 - b) + x3), dim)
    return y.reshape(x.shape)


def _quantize(x, fmt, rotation):
    """(packed codes, tiled block scales, row scales) of rows of finite values."""
    rows, k = x.shape
    block = BLOCK[fmt]
    v = _rotate(x.float()) if rotation else x.float()
    v = v.view(rows, k // block, block)
    amax = v.abs().amax(2)
    if fmt == "nvfp4":
        # 2688 = 6 * 448, the largest element times the largest block scale.
        mantissa, exponent = torch.frexp(amax.amax(1) / amax.new_tensor(2688.0))
        exponent = torch.where(mantissa > 0.5, exponent, exponent - 1).clamp_min(-126)
        row = torch.where(mantissa == 0, torch.ones_like(mantissa), torch.ldexp(torch.ones_like(mantissa), exponent))
        v = v / row.view(rows, 1, 1)
        # Divisors are tensors: a product with a rounded reciprocal would not keep the ties.
        scale = (amax / row.view(rows, 1) / amax.new_tensor(6.0)).to(torch.float8_e4m3fn)
        divisor = scale.float()
    else:
        row = torch.ones(rows, device=x.device)
        exponent = torch.where(amax == 0, -127, torch.frexp(amax)[1] - 3).clamp_min(-127)
        scale = (exponent + 127).to(torch.uint8)
        divisor = torch.ldexp(torch.ones_like(amax, dtype=torch.float64), exponent).float()
    live = (divisor != 0).unsqueeze(2)
    q = v / torch.where(live, divisor.unsqueeze(2), torch.ones_like(v[..., :1]))
    a = q.abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    code = torch.where(live, code, torch.zeros_like(code)) + 8 * torch.signbit(q)
    code = code.view(rows, k)
    packed = code[:, 0::2] + 16 * code[:, 1::2]
    return packed.to(torch.uint8), _tiles(scale.view(torch.uint8)).view(SCALE_TYPE[fmt]), row.view(rows, 1)


def _values(packed, tiles, fmt, kind=torch.float32):
    """What codes and block scales stand for, without the row scale."""
    rows, half = packed.shape
    k, block = 2 * half, BLOCK[fmt]
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=packed.device, dtype=kind)
    table = torch.cat((table, -table))
    code = torch.stack((packed & 15, packed >> 4), 2).view(rows, k)
    scale = _untile(tiles, rows, k // block).contiguous().view(SCALE_TYPE[fmt]).to(kind)
    return (table[code.int()].view(rows, k // block, block) * scale.unsqueeze(2)).view(rows, k)


# ---------------------------------------------------------------------------------------- inputs
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _normal(shape, g, scale=1.0):
    return torch.randn(shape, generator=g, device="cuda") * scale


def _activations(rows, k, g):
    """Rows of different sizes with a few strong channels, as a transformer's residual stream has them."""
    x = _normal((rows, k), g)
    x *= torch.exp(_normal((rows, 1), g, 0.5))
    strong = torch.randint(0, k, (max(1, k // 128),), generator=g, device="cuda")
    x[:, strong] *= 8.0
    return x


def _weights(n, k, g, fmt, rotation):
    w = _normal((n, k), g, k ** -0.5).bfloat16()
    return _quantize(w, fmt, rotation)


def prepare(case, seed):
    g = _generator(seed)
    op = case["op"]
    s = {"case": case}
    if op == "layer_norm":
        kind, weight = TYPES[case["type"]], TYPES[case["weight"]]
        rows, hidden = case["rows"], case["hidden"]
        s["x"] = (_activations(rows, hidden, g) + 0.25).to(kind)
        s["weight"] = (1.0 + _normal((hidden,), g, 0.1)).to(weight)
        s["bias"] = _normal((hidden,), g, 0.1).to(weight)
        if case["train"]:
            s["grad"] = _normal((rows, hidden), g).to(kind)
            for name in ("x", "weight", "bias"):
                s[name].requires_grad_(True)
    elif op == "quantize":
        s["x"] = _activations(case["rows"], case["k"], g).to(TYPES[case["type"]])
    elif op == "linear":
        m, n, k, fmt = case["m"], case["n"], case["k"], case["format"]
        s["a"] = _quantize(_activations(m, k, g).bfloat16(), fmt, 0)
        s["w"] = _weights(n, k, g, fmt, 0)
        s["bias"] = _normal((n,), g, 0.1) if case["bias"] else None
    else:
        m, n, k, fmt = case["m"], case["n"], case["k"], case["format"]
        s["grad"] = _normal((m, n), g).bfloat16()
        s["w"] = _weights(n, k, g, fmt, case["rotation"])
    return s


# ---------------------------------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        import comfyui_turing_utils_kernel as k
    if op == "layer_norm":
        x, weight, bias = state["x"], state["weight"], state["bias"]
        if own:
            y = k.turing_layer_norm(x, weight, bias, EPSILON)
            if not case["train"]:
                return {"y": y}
            dx, dw, db = torch.autograd.grad(y, (x, weight, bias), state["grad"])
            return {"y": y.detach(), "dx": dx, "dweight": dw, "dbias": db}
        with torch.no_grad():
            v, w = x.float(), weight.float()
            centred = v - v.mean(1, keepdim=True)
            rstd = 1.0 / torch.sqrt((centred * centred).mean(1, keepdim=True) + EPSILON)
            normal = centred * rstd
            y = (normal * w + bias.float()).to(x.dtype)
            if not case["train"]:
                return {"y": y}
            grad = state["grad"].float()
            g = grad * w
            dx = rstd * (g - g.mean(1, keepdim=True) - normal * (g * normal).mean(1, keepdim=True))
            return {"y": y, "dx": dx.to(x.dtype), "dweight": (grad * normal).sum(0).to(weight.dtype),
                    "dbias": grad.sum(0).to(bias.dtype)}
    fmt = case["format"]
    if op == "quantize":
        if own:
            codes, scale, row = k.turing_fp4_quantize(state["x"], fmt, case["rotation"])
            return {"values": k.turing_fp4_dequantize(codes, scale, row), "block_scale": scale, "row_scale": row}
        codes, scale, row = _quantize(state["x"], fmt, case["rotation"])
        return {"values": (_values(codes, scale, fmt) * row).bfloat16(), "block_scale": scale, "row_scale": row}
    w, w_scale, w_row = state["w"]
    if op == "linear":
        a, a_scale, a_row = state["a"]
        if own:
            return {"out": k.turing_fp4_linear(a, w, a_scale, w_scale, a_row, w_row, state["bias"])}
        out = _values(a, a_scale, fmt) @ _values(w, w_scale, fmt).t()
        out = out * a_row * w_row.view(1, -1)
        return {"out": (out if state["bias"] is None else out + state["bias"]).bfloat16()}
    if own:
        return {"dx": k.turing_fp4_linear_grad_input(state["grad"], w, w_scale, w_row, case["rotation"])}
    dx = state["grad"].float() @ (_values(w, w_scale, fmt) * w_row)
    return {"dx": (_rotate(dx) if case["rotation"] else dx).bfloat16()}


def work(case):
    """Bytes of inputs and outputs, and the operations of the definition."""
    op = case["op"]
    if op == "layer_norm":
        each = 2 if case["type"] != "fp32" else 4
        values = case["rows"] * case["hidden"]
        vectors = case["hidden"] * (2 if case["weight"] != "fp32" else 4)
        if case["train"]:
            return {"bytes": 4 * values * each + 4 * vectors, "flops": 20 * values}
        return {"bytes": 2 * values * each + 2 * vectors, "flops": 8 * values}
    block = BLOCK[case["format"]]
    if op == "quantize":
        values = case["rows"] * case["k"]
        return {"bytes": 4 * values + values // block + 4 * case["rows"], "flops": (14 if case["rotation"] else 4) * values}
    m, n, k = case["m"], case["n"], case["k"]
    weights = n * k // 2 + n * k // block + 4 * n
    if op == "linear":
        bias = 4 * n if case["bias"] else 0
        return {"bytes": weights + m * k // 2 + m * k // block + 4 * m + bias + 2 * m * n, "flops": 2 * m * n * k}
    return {"bytes": weights + 2 * m * n + 2 * m * k, "flops": 2 * m * n * k + (10 * m * k if case["rotation"] else 0)}


# ---------------------------------------------------------------------------------------- 64 bits
_SIGNS = [[1, 1, 1, -1], [1, 1, -1, 1], [1, -1, 1, 1], [-1, 1, 1, 1]]


def _exact_rotation(v):
    h = torch.tensor(_SIGNS, dtype=torch.float64, device=v.device) / 2
    h2 = torch.kron(h, h)
    return (v.reshape(-1, 256) @ torch.kron(h2, h2)).reshape(v.shape)


def _floor_log2(v):
    """Exponents from the bits: a logarithm may end beside a power of two."""
    return (v.double().view(torch.int64) >> 52) - 1023


def _nearest(v, grid):
    """Nearest grid value in 64 bits, ties to the even place in the grid."""
    a = v.abs()
    high = torch.searchsorted(grid, a).clamp(1, grid.numel() - 1)
    low = high - 1
    below, above = a - grid[low], grid[high] - a
    up = (above < below) | ((above == below) & (high % 2 == 0))
    return torch.where(up, grid[high], grid[low]) * torch.sign(v)


def _exact_quantize(x, fmt, rotation):
    v = x.double()
    if rotation:
        v = _exact_rotation(v)
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=v.device)
    blocks = v.view(v.shape[0], -1, BLOCK[fmt])
    peak = blocks.abs().amax(2)
    row = torch.ones((v.shape[0], 1), dtype=torch.float64, device=v.device)
    if fmt == "nvfp4":
        top = peak.amax(1, keepdim=True)
        power = (_floor_log2(top / 1.3125) - 11).double()
        power = (power + (torch.exp2(power) * 2688.0 < top)).clamp_min(-126)
        row = torch.where(top > 0, torch.exp2(power), row)
        e4m3 = torch.tensor([m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)][:-1],
                            dtype=torch.float64, device=v.device)
        scale = _nearest((peak / row / 6.0).clamp_max(448.0), e4m3)
        blocks = blocks / row.unsqueeze(2)
    else:
        scale = torch.exp2((_floor_log2(peak) - 2).clamp_min(-127).double())
    safe = torch.where(scale == 0, torch.ones_like(scale), scale).unsqueeze(2)
    values = _nearest((blocks / safe).clamp(-6, 6), grid) * scale.unsqueeze(2) * row.unsqueeze(2)
    rows, count = scale.shape
    mt, kt = -(-rows // 128), -(-count // 4)
    tiles = torch.full((mt * 128, kt * 4), 0.0 if fmt == "nvfp4" else 2.0 ** -127, dtype=torch.float64, device=v.device)
    tiles[:rows, :count] = scale
    tiles = tiles.view(mt, 4, 32, kt, 4).permute(0, 3, 2, 1, 4).reshape(mt, kt, 32, 16)
    return values.view(v.shape), tiles, row


def _exact_operand(operand, fmt):
    packed, tiles, row = operand
    low, high = (packed & 15).long(), (packed >> 4).long()
    code = torch.empty((packed.shape[0], 2 * packed.shape[1]), dtype=torch.long, device=packed.device)
    code[:, 0::2], code[:, 1::2] = low, high
    e, m = (code >> 1) & 3, code & 1
    value = torch.where(e == 0, 0.5 * m, (1 + 0.5 * m) * torch.exp2((e - 1).double())) * (1 - 2 * (code >> 3))
    r = torch.arange(code.shape[0], device=code.device).view(-1, 1)
    b = torch.arange(code.shape[1], device=code.device).view(1, -1) // BLOCK[fmt]
    bits = tiles.view(torch.uint8)[r // 128, b // 4, r % 32, 4 * (r % 128 // 32) + b % 4].double()
    if fmt == "nvfp4":
        e, m = torch.floor(bits / 8), bits % 8
        scale = torch.where(e == 0, m * 2.0 ** -9, (8 + m) * torch.exp2(e - 10))
    else:
        scale = torch.exp2(bits - 127)
    return value * scale * row.double().view(-1, 1)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    with torch.no_grad():
        if op == "layer_norm":
            x, w, b = s["x"].double(), s["weight"].double(), s["bias"].double()
            var, mean = torch.var_mean(x, 1, unbiased=False, keepdim=True)
            normal = (x - mean) / torch.sqrt(var + EPSILON)
            out = {"y": torch.addcmul(b, normal, w)}
            if case["train"]:
                grad = s["grad"].double()
                n = case["hidden"]
                through = grad * w
                a = through.sum(1, keepdim=True)
                c = torch.einsum("rh,rh->r", through, normal).view(-1, 1)
                out["dx"] = (n * through - a - normal * c) / (n * torch.sqrt(var + EPSILON))
                out["dweight"] = torch.einsum("rh,rh->h", grad, normal)
                out["dbias"] = grad.sum(0)
            return out
        if op == "quantize":
            values, tiles, row = _exact_quantize(s["x"], case["format"], case["rotation"])
            return {"values": values, "block_scale": tiles, "row_scale": row}
        w = _exact_operand(s["w"], case["format"])
        if op == "linear":
            out = torch.mm(_exact_operand(s["a"], case["format"]), w.t())
            return {"out": out if s["bias"] is None else out + s["bias"].double()}
        dx = torch.mm(s["grad"].double(), w)
        return {"dx": _exact_rotation(dx) if case["rotation"] else dx}
