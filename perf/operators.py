"""Measured calls: products of 8-bit integers with a scale per token and per channel, and the kernels that make their operands.

A pass is ONE call of one operator, as a layer with 8-bit weights makes it:

* "norm": residual <- x + residual, the RMS norm of the sum, and the normed rows in 8 bits with a scale per row;
* "act": act(gate) * up of rows [gate | up], in 8 bits with a scale per row;
* "quantize": rows as they are, in 8 bits with a scale per row (an attention's output in front of its projection, a weight's rows);
* "linear": the product of 8-bit rows with an 8-bit weight, scaled per row and per column, with or without a bias.

A scale is the largest magnitude of its row over 127, an element is held as its nearest whole multiple.  What is held in 8 bits is
returned as the values it stands for, in the type of the rows it was made of (32-bit rows: in bfloat16, which holds more than they do).

Sizes are those of the benchmark's models (widths of 4,096 and 5,120, feed-forwards of 12,288 and 25,600), and ragged ones.
"""

import math

import torch

own = False  # False: the operators in elementary 32-bit operations; True: the framework's kernels

_TYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
_BYTES = {"bfloat16": 2, "float16": 2, "float32": 4}
_EPS = 1e-6


# ---------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------
def listed():
    return [
        # the norm in front of a layer's products: eight requests decoding; a prompt; a ragged float16 prompt, first layer (no residual)
        dict(name="norm_decode", op="norm", rows=8, cols=4096, dtype="bfloat16", residual=True),
        dict(name="norm_prompt", op="norm", rows=2048, cols=4096, dtype="bfloat16", residual=True),
        dict(name="norm_ragged", op="norm", rows=1023, cols=5120, dtype="float16", residual=False),
        # the gated activation in front of a feed-forward's second product: sixteen requests decoding; a prompt of the widest model
        dict(name="act_decode", op="act", rows=16, cols=12288, dtype="bfloat16", act="silu"),
        dict(name="act_prompt", op="act", rows=2048, cols=25600, dtype="bfloat16", act="silu"),
        # an attention's output in front of its projection: one request decoding; a ragged prompt whose rows lie in wider ones
        dict(name="quantize_single", op="quantize", rows=1, cols=4096, dtype="bfloat16", wider=0),
        dict(name="quantize_prompt", op="quantize", rows=2047, cols=8192, dtype="bfloat16", wider=2048),
        # products: q, k and v for one request; gate and up for eight; down for a batch of 64; gate and up for a prompt; a ragged
        # prompt with a bias and a 32-bit result, whose k ends inside a tile (rows padded to 16 bytes)
        dict(name="linear_single", op="linear", rows=1, cols=6144, k=4096, dtype="bfloat16", bias=False),
        dict(name="linear_decode", op="linear", rows=8, cols=24576, k=4096, dtype="bfloat16", bias=False),
        dict(name="linear_batch", op="linear", rows=64, cols=4096, k=12288, dtype="bfloat16", bias=False),
        dict(name="linear_prompt", op="linear", rows=2048, cols=24576, k=4096, dtype="bfloat16", bias=False),
        dict(name="linear_ragged", op="linear", rows=333, cols=2057, k=1100, dtype="float32", bias=True),
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _size(rng, lo, hi):
    """A width: a multiple of 64 in three cases of four, else any number."""
    n = _log(rng, lo, hi)
    return n if rng.random() < 0.25 else max(64, n // 64 * 64)


def draw(rng):
    op = rng.choice(("norm", "act", "quantize", "linear", "linear"))
    dtype = rng.choice(("bfloat16", "bfloat16", "float16", "float32"))
    if op == "linear":
        cols, k = _size(rng, 64, 24576), _size(rng, 64, 12288)
        rows = _log(rng, 1, max(1, min(2048, 2048 * 24576 * 4096 // (cols * k))))
        return dict(op=op, rows=rows, cols=cols, k=k, dtype=dtype, bias=rng.random() < 0.3)
    cols = _size(rng, 64, 25600 if op == "act" else 8192)
    rows = _log(rng, 1, 2048)
    case = dict(op=op, rows=rows, cols=cols, dtype=dtype)
    if op == "norm":
        case["residual"] = rng.random() < 0.75
    elif op == "act":
        case["act"] = rng.choice(("silu", "gelu_tanh"))
    else:
        case["wider"] = rng.choice((0, 0, 64, 1000))
    return case


def work(case):
    rows, cols, size = case["rows"], case["cols"], _BYTES[case["dtype"]]
    n = rows * cols
    if case["op"] == "norm":
        return {"bytes": n * (size * (3 if case["residual"] else 1) + 1) + 4 * (rows + cols), "flops": 6 * n}
    if case["op"] == "act":
        return {"bytes": n * (2 * size + 1) + 4 * rows, "flops": 8 * n}
    if case["op"] == "quantize":
        return {"bytes": n * (size + 1) + 4 * rows, "flops": 3 * n}
    k = case["k"]
    return {"bytes": (rows + cols) * (k + 4) + n * size + (cols * size if case["bias"] else 0), "flops": 2 * n * k}


# ---------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------
class State:
    pass


def _rows(g, rows, cols, dtype, spread=0.5):
    """Activations: rows of unequal size, and one channel in 256 that is ten times the others."""
    x = torch.randn(rows, cols, generator=g, device="cuda")
    x *= torch.exp(spread * torch.randn(rows, 1, generator=g, device="cuda"))
    x *= 1 + 9 * (torch.rand(cols, generator=g, device="cuda") < 1 / 256)
    return x.to(dtype)


def _padded(rows, cols):
    """8-bit rows on borders of 16 bytes."""
    return torch.zeros(rows, -(-cols // 16) * 16, dtype=torch.int8, device="cuda")[:, :cols]


def _held(x):
    """(8-bit rows, scales) of x: what a program has in hand in front of a product."""
    scales = x.abs().amax(1) / 127
    q = _padded(*x.shape)
    q.copy_(torch.round(x / scales[:, None]))
    return q, scales


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = State()
    s.op, s.dtype, s.act = case["op"], _TYPES[case["dtype"]], case.get("act")
    rows, cols = case["rows"], case["cols"]
    if s.op == "linear":
        s.x, s.x_scales = _held(_rows(g, rows, case["k"], torch.float32))
        s.w, s.w_scales = _held(torch.randn(cols, case["k"], generator=g, device="cuda").mul_(0.02))
        s.bias = (0.1 * torch.randn(cols, generator=g, device="cuda")).to(s.dtype) if case["bias"] else None
        s.out = torch.empty(rows, cols, dtype=s.dtype, device="cuda")
        return s
    if s.op == "norm":
        s.x = _rows(g, rows, cols, s.dtype)
        s.residual = _rows(g, rows, cols, s.dtype) if case["residual"] else None
        s.weight = 1 + 0.2 * torch.randn(cols, generator=g, device="cuda")
    elif s.op == "act":
        s.x = _rows(g, rows, 2 * cols, s.dtype)
    else:
        wide = cols + case["wider"]
        s.x = _rows(g, rows, wide, s.dtype)[:, :cols]
    s.q, s.scales = _padded(rows, cols), torch.empty(rows, device="cuda")
    s.values = torch.empty(rows, cols, dtype=torch.bfloat16 if s.dtype == torch.float32 else s.dtype, device="cuda")
    return s


# ---------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------
def _plain_quantize(y):
    """(the values that the 8-bit rows stand for, scales) of 32-bit rows."""
    scales = y.abs().amax(1) / 127
    q = torch.round(y / scales[:, None].clamp_min(1e-37)).to(torch.int8)
    return q, scales


def _answer(s):
    torch.mul(s.q, s.scales[:, None], out=s.values)  # the values that the 8-bit rows stand for, rounded once
    out = {"values": s.values, "scales": s.scales}
    if s.op == "norm" and s.residual is not None:
        out["residual"] = s.residual
    return out


def _run_plain(s):
    if s.op == "linear":
        y = (s.x.float() @ s.w.float().t()) * s.x_scales[:, None] * s.w_scales
        if s.bias is not None:
            y = y + s.bias.float()
        s.out.copy_(y)
        return s.out
    if s.op == "norm":
        y = s.x.float()
        if s.residual is not None:
            y = y + s.residual.float()
            s.residual.copy_(y)
        y = y * torch.rsqrt((y * y).mean(1, keepdim=True) + _EPS) * s.weight
    elif s.op == "act":
        gate, up = s.x.float().chunk(2, dim=1)
        if s.act == "silu":
            y = gate / (1 + torch.exp(-gate)) * up
        else:
            y = 0.5 * gate * (1 + torch.tanh(math.sqrt(2 / math.pi) * (gate + 0.044715 * gate * gate * gate))) * up
    else:
        y = s.x.float()
    q, scales = _plain_quantize(y)
    s.q.copy_(q)
    s.scales.copy_(scales)
    return _answer(s)


def _run_own(s):
    from ullm_b200.csrc import kernels

    K = kernels()
    if s.op == "linear":
        return K.linear_int8(s.x, s.x_scales, s.w, s.w_scales, s.out, s.bias)
    if s.op == "norm":
        K.add_rmsnorm_int8(s.x, s.residual, s.weight, _EPS, s.q, s.scales)
    elif s.op == "act":
        K.act_mul_int8(s.x, s.q, s.scales, 0 if s.act == "silu" else 1)
    else:
        K.quantize_rows_int8(s.x, s.q, s.scales)
    return _answer(s)


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if s.op == "linear":
        total = torch.empty(case["rows"], case["cols"], dtype=torch.float64, device="cuda")
        torch.mm(s.x.double(), s.w.double().t(), out=total)
        total.mul_(s.w_scales.double()).mul_(s.x_scales.double().unsqueeze(1))
        return total if s.bias is None else total.add_(s.bias.double())
    out = {}
    x = s.x.double()
    if s.op == "norm":
        if s.residual is not None:
            x = x + s.residual.double()
            out["residual"] = x
        mean = x.pow(2).sum(1, keepdim=True) / case["cols"]
        x = x / (mean + _EPS).sqrt() * s.weight.double()
    elif s.op == "act":
        gate, up = x[:, :case["cols"]], x[:, case["cols"]:]
        if s.act == "silu":
            x = gate * torch.sigmoid(gate) * up
        else:  # (1 + tanh v) / 2 = 1 / (1 + exp(-2 v))
            x = gate * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (gate + 0.044715 * gate.pow(3))) * up
    largest = x.abs().max(1).values
    out["scales"] = largest / 127
    step = out["scales"].unsqueeze(1)
    out["values"] = torch.where(step > 0, torch.round(x / step) * step, 0.0)
    return out
