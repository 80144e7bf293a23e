"""The cases on which the 8-bit block-scaled dense operators are measured.

One number format runs through all of them: 8-bit elements with one power-of-two scale for every block of 128
columns of a row (or of 128 x 128 elements), held as its biased exponent byte (the scale is 2^(byte - 127)). The
operators are the quantizer to 8-bit floating point, the matrix product of two such operands, the INT8 checkpoint of
an activation function's input, that function's gradient from the checkpoint, and the weight gradient of a linear
layer whose input was kept as such a checkpoint.
"""
import math

import torch

own = False

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16,
         "e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2, "e4m3": 1, "e5m2": 1}
LARGEST = {"e4m3": 448.0, "e5m2": 57344.0, "int8": 127.0}
BLOCK = 128


def listed():
    return [
        # The aggregated features of a million nodes (a graph layer's SpMM writes them in fp32), made ready for the product.
        {"name": "quantize_nodes", "op": "quantize", "rows": 1048576, "cols": 128, "type": "fp32", "to": "e4m3", "block_rows": 1},
        # A layer's weights after an optimizer step; the last blocks end inside the matrix.
        {"name": "quantize_weight", "op": "quantize", "rows": 4000, "cols": 4100, "type": "bf16", "to": "e4m3", "block_rows": 128},
        # One token, or one queried node, through a layer: latency and the weights' bytes.
        {"name": "product_token", "op": "product", "m": 1, "n": 4096, "k": 4096, "a": "e4m3", "layout": "nk", "out": "bf16", "bias": False},
        # A training step's forward product.
        {"name": "product_layer", "op": "product", "m": 8192, "n": 4096, "k": 4096, "a": "e4m3", "layout": "nk", "out": "bf16", "bias": False},
        # Node features through a narrow layer: many rows, one tile of columns, an output of four times the input's width.
        {"name": "product_nodes", "op": "product", "m": 1048576, "n": 128, "k": 256, "a": "e4m3", "layout": "nk", "out": "fp32", "bias": True},
        # The gradient of a layer's input: e5m2 gradients times the layer's weights, contracted over the weights' rows; odd sizes.
        {"name": "product_input_grad", "op": "product", "m": 4001, "n": 2000, "k": 4100, "a": "e5m2", "layout": "kn", "out": "bf16", "bias": False},
        # An activation function of a training step, its input kept for the backward pass.
        {"name": "checkpoint_gelu", "op": "checkpoint", "rows": 8192, "cols": 4096, "type": "bf16", "activation": "gelu"},
        # The same for few rows of an odd width.
        {"name": "checkpoint_odd", "op": "checkpoint", "rows": 333, "cols": 1001, "type": "fp32", "activation": "silu"},
        # Its backward pass from the checkpoint.
        {"name": "backward_gelu", "op": "backward", "rows": 8192, "cols": 4096, "type": "bf16", "activation": "gelu"},
        # A graph layer's gradient through its activation, over all nodes.
        {"name": "backward_nodes", "op": "backward", "rows": 1048576, "cols": 128, "type": "fp32", "activation": "relu"},
        # The weight gradient of a training step.
        {"name": "weight_grad_layer", "op": "weight_grad", "rows": 8192, "n": 4096, "k": 2048, "type": "bf16"},
        # The weight gradient of a graph layer: one small matrix, a sum over all nodes.
        {"name": "weight_grad_nodes", "op": "weight_grad", "rows": 1048576, "n": 128, "k": 256, "type": "fp32"},
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _width(rng, low, high):
    """A width: as often as not a multiple of 128, else any, odd ones among them."""
    w = _spread(rng, low, high)
    return w if w < 128 or rng.random() < 0.5 else w // 128 * 128


def draw(rng):
    op = rng.choice(["quantize", "product", "product", "checkpoint", "backward", "weight_grad"])
    if op == "product":
        n, k = _width(rng, 16, 8192), _width(rng, 16, 8192)
        most = min(1048576, int(2.0 ** 37 / (n * k)), int(1.4e9 / (k + 4 * n)))
        layout = rng.choice(["nk", "nk", "kn"])
        return {"op": op, "m": _spread(rng, 1, max(1, most)), "n": n, "k": k, "a": rng.choice(["e4m3", "e4m3", "e5m2"]),
                "layout": layout, "out": rng.choice(["bf16", "fp16", "fp32"]), "bias": rng.random() < 0.5}
    if op == "weight_grad":
        n, k = _width(rng, 16, 8192), _width(rng, 16, 8192)
        most = min(1048576, int(2.0 ** 36 / (n * k)), int(1.2e9 / (k + 4 * n)))
        return {"op": op, "rows": _spread(rng, 1, max(1, most)), "n": n, "k": k, "type": rng.choice(["fp32", "bf16", "bf16", "fp16"])}
    cols = _width(rng, 16, 8192)
    rows = _spread(rng, 1, min(1048576, 2 ** 25 // cols))
    kind = rng.choice(["fp32", "bf16", "bf16", "fp16"])
    if op == "quantize":
        return {"op": op, "rows": rows, "cols": cols, "type": kind, "to": rng.choice(["e4m3", "e4m3", "e5m2"]), "block_rows": rng.choice([1, 128])}
    return {"op": op, "rows": rows, "cols": cols, "type": kind, "activation": rng.choice(["relu", "gelu", "gelu_tanh", "silu"])}


def _ceil(a, b):
    return -(-a // b)


def _values(gen, rows, cols, scale, dtype):
    """Rows of normal values of differing sizes, some columns far larger, the last rows (padding) zero."""
    x = torch.randn(rows, cols, device="cuda", generator=gen)
    x *= torch.exp(0.7 * torch.randn(rows, 1, device="cuda", generator=gen)) * scale
    x *= torch.where(torch.rand(1, cols, device="cuda", generator=gen) < 0.01, 20.0, 1.0)
    if rows > 16:
        x[rows - rows // 16:] = 0
    return x.to(dtype)


def _with_stride(q):
    """The same values with rows that begin on 16 bytes, as a program lays its 8-bit operands out."""
    rows, cols = q.shape
    whole = torch.zeros(rows, _ceil(cols, 16) * 16, dtype=torch.uint8, device=q.device)
    whole[:, :cols] = q.view(torch.uint8)
    return whole.view(q.dtype)[:, :cols]


def _blocks(x, block_rows):
    """x cut into its blocks, [row block, row, column block, column], zeros behind its ends."""
    rows, cols = x.shape
    rb, cb = _ceil(rows, block_rows), _ceil(cols, BLOCK)
    if (rows, cols) != (rb * block_rows, cb * BLOCK):
        x = torch.nn.functional.pad(x, (0, cb * BLOCK - cols, 0, rb * block_rows - rows))
    return x.reshape(rb, block_rows, cb, BLOCK)


def _unblock(x, rows, cols):
    return x.reshape(x.shape[0] * x.shape[1], -1)[:rows, :cols]


def _power(e):
    """2^e in 32 bits, by its bits: -126 <= e <= 127."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _exponents(x, block_rows, largest):
    """Each block's exponent: the least e with absmax <= 2^e * largest, 0 for a block of zeros."""
    top = _blocks(x, block_rows).abs().amax(dim=(1, 3))
    fraction, e = torch.frexp(top / largest)  # top / largest = fraction * 2^e, fraction in [0.5, 1)
    e = torch.where(fraction == 0.5, e - 1, e)
    e = torch.where(_power(e.clamp(-126, 119)) * largest < top, e + 1, e)  # the division's rounding
    return torch.where(top == 0, torch.zeros_like(e), e.clamp(min=-126))


def _quantize(x, block_rows, kind):
    """(q, scale bytes) of x in 32 bits."""
    x = x.float()
    e = _exponents(x, block_rows, LARGEST[kind])
    v = _unblock(_blocks(x, block_rows) * _power(-e)[:, None, :, None], *x.shape)
    q = v.round().to(torch.int8) if kind == "int8" else v.to(TYPES[kind])
    return q, (e + 127).to(torch.uint8)


def _restore(q, scales, block_rows=1):
    """The values that q and its scale bytes stand for, in 32 bits (exact)."""
    s = _power(scales.int() - 127)
    return _unblock(_blocks(q.float(), block_rows) * s[:, None, :, None], *q.shape)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    op, state = case["op"], dict(case)

    def empty(rows, cols, dtype):
        return torch.empty(rows, cols, dtype=dtype, device="cuda")

    if op == "product":
        m, n, k = case["m"], case["n"], case["k"]
        a, state["a_scales"] = _quantize(_values(gen, m, k, 1.0 if case["a"] == "e4m3" else 1e-3, torch.bfloat16), 1, case["a"])
        w = torch.randn((n, k) if case["layout"] == "nk" else (k, n), device="cuda", generator=gen) / math.sqrt(k)
        b, state["b_scales"] = _quantize(w.to(torch.bfloat16), BLOCK, "e4m3")
        state["a_data"], state["b_data"] = _with_stride(a), _with_stride(b)
        state["bias_data"] = torch.randn(n, device="cuda", generator=gen) if case["bias"] else None
        state["output"] = empty(m, n, TYPES[case["out"]])
        return state
    if op == "weight_grad":
        dtype = TYPES[case["type"]]
        x = _values(gen, case["rows"], case["k"], 1.0, torch.bfloat16 if dtype != torch.float32 else dtype)
        q, state["scales"] = _quantize(x, 1, "int8")
        state["q"] = _with_stride(q)
        state["grad_y"] = _values(gen, case["rows"], case["n"], 1e-2, dtype)
        state["grad_w"] = empty(case["n"], case["k"], torch.float32)
        return state
    rows, cols, dtype = case["rows"], case["cols"], TYPES[case["type"]]
    x = _values(gen, rows, cols, 1.0, dtype)
    if op == "backward":
        q, state["scales"] = _quantize(x, 1, "int8")
        state["q"] = _with_stride(q)
        state["grad_y"] = _values(gen, rows, cols, 1e-2, dtype)
        state["grad_x"] = empty(rows, cols, dtype)
        return state
    state["x"] = x
    block_rows = case.get("block_rows", 1)
    held = TYPES[case["to"]] if op == "quantize" else torch.int8
    state["q"] = _with_stride(torch.zeros(rows, cols, dtype=torch.uint8, device="cuda").view(held))
    state["scales"] = torch.zeros(_ceil(rows, block_rows), _ceil(cols, BLOCK), dtype=torch.uint8, device="cuda")
    if op == "checkpoint":
        state["y"] = empty(rows, cols, dtype)
    return state


def _activation(x, kind):
    if kind == "relu":
        return torch.clamp(x, min=0)
    if kind == "silu":
        return x / (1 + torch.exp(-x))
    if kind == "gelu":
        return x * 0.5 * torch.erfc(-x * math.sqrt(0.5))
    u = math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)
    return 0.5 * x * (1 + torch.tanh(u))


def _slope(x, kind):
    """The derivative of an activation function."""
    if kind == "relu":
        return (x > 0).to(x.dtype)
    if kind == "silu":
        s = 1 / (1 + torch.exp(-x))
        return s * (1 + x * (1 - s))
    if kind == "gelu":
        return 0.5 * torch.erfc(-x * math.sqrt(0.5)) + x * torch.exp(-0.5 * x * x) * (1 / math.sqrt(2 * math.pi))
    t = torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3))
    return 0.5 * (1 + t) + 0.5 * x * (1 - t * t) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * x * x)


def _plain(s):
    op = s["op"]
    if op == "quantize":
        return _quantize(s["x"], s["block_rows"], s["to"])
    if op == "product":
        a = _restore(s["a_data"], s["a_scales"])
        b = _restore(s["b_data"], s["b_scales"], BLOCK)
        y = a @ (b.t() if s["layout"] == "nk" else b)
        if s["bias_data"] is not None:
            y = y + s["bias_data"]
        return y.to(TYPES[s["out"]])
    if op == "checkpoint":
        q, scales = _quantize(s["x"], 1, "int8")
        return _activation(s["x"].float(), s["activation"]).to(s["x"].dtype), q, scales
    if op == "backward":
        return (s["grad_y"].float() * _slope(_restore(s["q"], s["scales"]), s["activation"])).to(s["grad_y"].dtype)
    return s["grad_y"].float().t() @ _restore(s["q"], s["scales"])


def _own(s):
    import tcc_spmm_b200 as T

    op = s["op"]
    if op == "quantize":
        T.quantize_blocks_fp8(s["x"], s["q"], s["scales"], block_rows=s["block_rows"])
        return s["q"], s["scales"]
    if op == "product":
        T.matmul_fp8_blocks(s["a_data"], s["a_scales"], s["b_data"], s["b_scales"], s["output"], bias=s["bias_data"],
                            b_layout=s["layout"])
        return s["output"]
    if op == "checkpoint":
        T.activation_checkpoint_int8(s["x"], s["y"], s["q"], s["scales"], activation=s["activation"])
        return s["y"], s["q"], s["scales"]
    if op == "backward":
        T.activation_backward_int8(s["grad_y"], s["q"], s["scales"], s["grad_x"], activation=s["activation"])
        return s["grad_x"]
    T.weight_grad_int8(s["grad_y"], s["q"], s["scales"], s["grad_w"])
    return s["grad_w"]


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    op = case["op"]
    if op == "product":
        m, n, k = case["m"], case["n"], case["k"]
        kb = _ceil(k, BLOCK)
        read = m * k + n * k + m * kb + _ceil(n, BLOCK) * kb + (4 * n if case["bias"] else 0)
        return {"bytes": read + m * n * SIZE[case["out"]], "flops": 2 * m * n * k}
    if op == "weight_grad":
        rows, n, k = case["rows"], case["n"], case["k"]
        return {"bytes": rows * (n * SIZE[case["type"]] + k + _ceil(k, BLOCK)) + 4 * n * k, "flops": 2 * rows * n * k}
    rows, cols, size = case["rows"], case["cols"], SIZE[case["type"]]
    count, scales = rows * cols, _ceil(rows, case.get("block_rows", 1)) * _ceil(cols, BLOCK)
    if op == "quantize":
        return {"bytes": count * (size + 1) + scales, "flops": 3 * count}
    return {"bytes": count * (2 * size + 1) + scales, "flops": 12 * count}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------


def _exact_power(e):
    """2^e in 64 bits, for whole e, by its bits."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _exact_scales(x, block_rows, largest):
    """Scale bytes by comparison: how many of the powers 2^-126, 2^-125, ... are too small for the block's absmax."""
    rows, cols = x.shape
    rb, cb = _ceil(rows, block_rows), _ceil(cols, BLOCK)
    top = torch.zeros(rb, cb, dtype=torch.float64, device=x.device)
    for c in range(cb):
        part = x[:, c * BLOCK:(c + 1) * BLOCK].abs().amax(dim=1).double()
        if block_rows == 1:
            top[:, c] = part
        else:
            top[:, c] = torch.stack([piece.max() for piece in part.split(block_rows)])
    powers = _exact_power(torch.arange(-126, 128, device=x.device)) * largest
    steps = torch.bucketize(top, powers)  # the first power that is not below absmax
    return torch.where(top == 0, torch.full_like(steps, 127), steps + 1)


def _exact_repeat(bytes_, block_rows, rows, cols):
    s = _exact_power(bytes_.long() - 127)
    return s.repeat_interleave(block_rows, 0)[:rows].repeat_interleave(BLOCK, 1)[:, :cols]


def _exact_quantize(x, block_rows, kind):
    bytes_ = _exact_scales(x, block_rows, LARGEST[kind])
    v = x.double() / _exact_repeat(bytes_, block_rows, *x.shape)
    if kind == "int8":
        return torch.round(v).to(torch.int8), bytes_.to(torch.uint8)
    kept, lowest = (3, -6) if kind == "e4m3" else (2, -14)  # bits behind the point, the least normal exponent
    step = _exact_power((torch.frexp(v)[1] - 1).clamp(min=lowest) - kept)
    return torch.round(v / step) * step, bytes_.to(torch.uint8)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "quantize":
        return _exact_quantize(s["x"], case["block_rows"], case["to"])
    if op == "product":
        m, n, k = case["m"], case["n"], case["k"]
        a = s["a_data"].double() * _exact_repeat(s["a_scales"], 1, m, k)
        b = s["b_data"].double() * _exact_repeat(s["b_scales"], BLOCK, *s["b_data"].shape)
        y = torch.matmul(a, b.t() if case["layout"] == "nk" else b)
        return y if s["bias_data"] is None else y + s["bias_data"].double()
    if op == "weight_grad":
        x = s["q"].double() * _exact_repeat(s["scales"], 1, case["rows"], case["k"])
        return torch.matmul(s["grad_y"].double().t(), x)
    kind = case["activation"]
    if op == "checkpoint":
        x = s["x"].double()
        if kind == "relu":
            y = torch.where(x > 0, x, torch.zeros_like(x))
        elif kind == "silu":
            y = x * torch.special.expit(x)
        elif kind == "gelu":
            y = x * torch.special.ndtr(x)
        else:
            y = x * torch.special.expit(2 * math.sqrt(2 / math.pi) * (x + 0.044715 * x * x * x))
        return (y,) + _exact_quantize(s["x"], 1, "int8")
    x = s["q"].double() * _exact_repeat(s["scales"], 1, case["rows"], case["cols"])
    if kind == "relu":
        slope = (x > 0).double()
    elif kind == "silu":
        slope = torch.special.expit(x) * (1 + x * torch.special.expit(-x))
    elif kind == "gelu":
        slope = torch.special.ndtr(x) + x * torch.exp(-x * x / 2) / math.sqrt(2 * math.pi)
    else:
        c = math.sqrt(2 / math.pi)
        p = torch.special.expit(2 * c * (x + 0.044715 * x * x * x))
        slope = p + x * p * (1 - p) * 2 * c * (1 + 3 * 0.044715 * x * x)
    return s["grad_y"].double() * slope
