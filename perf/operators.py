"""What the 4-bit matrices are timed on: quantisation, the product with 16-bit activations, the product of two 4-bit
operands and the gated feed-forward's front half.

A matrix in microscaled 4 bits (MXFP4) is two byte tensors.  `codes` [rows, K / 2] holds two e2m1 values a byte (element
2j in the low half; sign, then 0, 0.5, 1, 1.5, 2, 3, 4, 6), `scales` [rows, K / 32] one power of two for 32 neighbouring
values of a row (exponent + 127).  A block's exponent is the smallest with which nothing is cut off: max |x| <= 6 * 2^e.

A case is a dict of plain values; `prepare` makes what a serving program has in hand (activations, and a matrix that was
brought into 4 bits when the model was loaded), `run` does one call, `exact` gives the same results in 64 bits.  Sizes are those
of the OPT family and of the other decoders' benchmark configurations.

Kinds of cases:
  quantize    rows to 4 bits and back to the values that they then stand for (in bfloat16, which holds each exactly)
  linear      16-bit activations by a 4-bit matrix; bias, activation; with `residual` added to the 32-bit stream
  product     the activations are brought into 4 bits too: quantisation and the product of two 4-bit operands
  gated       act(gate) * up of a gated feed-forward, gate and up rows of one 4-bit matrix; `quantized`: the activations too
"""
import math

import torch

own = False

DEV = "cuda:0"
STD = 0.02                            # of every random matrix, as the family is initialised
TORCH = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # one token's activations on their way into a product of two 4-bit operands: two launches and nothing else
        dict(name="quantize_1x4096", kind="quantize", dtype="bfloat16", rows=1, width=4096),
        # a prompt's activations in a width that is no power of two
        dict(name="quantize_777x5120", kind="quantize", dtype="float16", rows=777, width=5120),
        # a feed-forward's matrix of the 6.7B sizes while a model is loaded
        dict(name="quantize_16384x4096", kind="quantize", dtype="bfloat16", rows=16384, width=4096),
        # one user's chat on the smallest model: queries, keys and values of one token
        dict(name="linear_b1_768", kind="linear", dtype="float16", tokens=1, width=768, out=2304, act="none", residual=False),
        # one user on a large model: the feed-forward's first matrix is streamed for a single token
        dict(name="linear_b1_4096", kind="linear", dtype="bfloat16", tokens=1, width=4096, out=16384, act="relu", residual=False),
        # a small batch through the 13B sizes' second feed-forward matrix, into the residual stream
        dict(name="linear_b13_20480", kind="linear", dtype="float16", tokens=13, width=20480, out=5120, act="none", residual=True),
        # a served step: a portion of a prompt beside decode tokens, 2.7B sizes
        dict(name="linear_481_2560", kind="linear", dtype="float16", tokens=481, width=2560, out=10240, act="relu", residual=False),
        # a long prompt through the 6.7B sizes' first feed-forward matrix
        dict(name="linear_2048_4096", kind="linear", dtype="bfloat16", tokens=2048, width=4096, out=16384, act="gelu_new", residual=False),
        # decode tokens of eight users with 4-bit activations: an output projection
        dict(name="product_b8_4096", kind="product", dtype="bfloat16", tokens=8, width=4096, out=4096, act="none", residual=False),
        # a long prompt with 4-bit activations
        dict(name="product_2048_4096", kind="product", dtype="bfloat16", tokens=2048, width=4096, out=16384, act="relu", residual=False),
        # one token through a gated feed-forward's front half
        dict(name="gated_b1_4096", kind="gated", dtype="bfloat16", tokens=1, width=4096, out=8192, act="silu", quantized=False),
        # a prompt through it, with 4-bit activations
        dict(name="gated_1531_4096", kind="gated", dtype="bfloat16", tokens=1531, width=4096, out=8192, act="silu", quantized=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["quantize", "linear", "linear", "product", "gated"])
    dtype = rng.choice(["bfloat16", "float16"])
    if kind == "quantize":
        # single tokens to whole matrices; rows of any length, so that last blocks are short
        rows, width = _log(rng, 1, 16384), _log(rng, 33, 20480)
        rows = max(1, min(rows, 16384 * 4096 // width))
        return dict(kind=kind, dtype=rng.choice(["bfloat16", "float16", "float32"]), rows=rows, width=width)
    tokens = _log(rng, 1, 2048)
    width = 32 * _log(rng, 16, 640)
    if kind == "gated":
        out = 8 * _log(rng, 64, 1024)
        if tokens * width * out > 2048 * 4096 * 8192:
            tokens = max(1, 2048 * 4096 * 8192 // (width * out))
        return dict(kind=kind, dtype=dtype, tokens=tokens, width=width, out=out, act=rng.choice(["silu", "gelu_new", "relu"]), quantized=rng.random() < 0.5)
    out = rng.choice([8 * _log(rng, 64, 2560), _log(rng, 500, 20480)])      # now and then a number of outputs that nothing divides
    if width * out > 4096 * 16384:
        out = 4096 * 16384 // width
    if tokens * width * out > 2048 * 4096 * 16384:
        tokens = max(1, 2048 * 4096 * 16384 // (width * out))
    return dict(kind=kind, dtype=dtype, tokens=tokens, width=width, out=out, act=rng.choice(["none", "relu", "gelu_new"]), residual=rng.random() < 0.3)


# ---- plain forms ---------------------------------------------------------------------------------------------------
def _to_blocks(x):
    """32-bit rows as blocks of 32, zeros behind the last value."""
    rows, width = x.shape
    blocks = -(-width // 32)
    x = torch.nn.functional.pad(x, (0, blocks * 32 - width))
    return x.view(rows, blocks, 32)


def _exponents(x):
    """The blocks' exponents: the smallest e with max |x| <= 6 * 2^e, from the bits of the largest value."""
    bits = x.abs().amax(-1).view(torch.int32)
    normal = (bits >> 23) - 129 + ((bits & 0x7FFFFF) > 0x400000).int()       # 1.5 * 2^2 is the largest that e = exponent - 2 holds
    return normal.clamp(-127, 127)


def _round_e2m1(v):
    """Rows of |v| <= 6 to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6, ties to the even code."""
    a = v.abs()
    q = torch.where(a < 2, (a * 2).round() * 0.5, torch.where(a < 4, a.round(), (a * 0.5).round() * 2))
    return torch.copysign(q, v)


def _times_power(x, e):
    """x * 2^e for whole e between -127 and 127, exactly: in two factors that are normal numbers."""
    half = e >> 1
    two = lambda n: ((n + 127) << 23).view(torch.float32)       # noqa: E731
    return x * two(half) * two(e - half)


def _quantized(x):
    """The values that rows stand for in 4 bits, as 32-bit blocks."""
    b = _to_blocks(x.float())
    e = _exponents(b).unsqueeze(-1)
    return _times_power(_round_e2m1(_times_power(b, -e)), e)


def _pack(x):
    """32-bit rows -> (codes, scales)."""
    b = _to_blocks(x)
    e = _exponents(b)
    q = _round_e2m1(_times_power(b, -e.unsqueeze(-1)))
    edges = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=x.device)
    code = torch.bucketize(q.abs(), edges).to(torch.uint8) + 8 * torch.signbit(q).to(torch.uint8)
    code = code.view(x.shape[0], -1)
    return code[:, 0::2] + (code[:, 1::2] << 4), (e + 127).to(torch.uint8)


def _unpack(codes, scales, width):
    table = torch.tensor(MAGNITUDES + tuple(-m for m in MAGNITUDES), device=codes.device)
    v = torch.stack((table[(codes & 15).int()], table[(codes >> 4).int()]), -1).view(codes.shape[0], -1, 32)
    return _times_power(v, scales.int().unsqueeze(-1) - 127).view(codes.shape[0], -1)[:, :width]


def _activation(x, name):
    if name == "relu":
        return torch.clamp(x, min=0)
    if name == "silu":
        return x / (1 + torch.exp(-x))
    if name == "gelu_new":
        return 0.5 * x * (1 + torch.tanh(0.7978845608028654 * (x + 0.044715 * x * x * x)))
    return x


# ---- cases ---------------------------------------------------------------------------------------------------------
def _activations(g, tokens, width, dtype):
    """Rows behind a norm: unit size, a few channels much larger than the rest, as trained decoders have them."""
    x = torch.randn(tokens, width, generator=g, device=DEV)
    x[:, torch.randint(0, width, (max(1, width // 256),), generator=g, device=DEV)] *= 12.0
    return x.to(TORCH[dtype])


def _inputs(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    if case["kind"] == "quantize":
        return dict(x=(torch.randn(case["rows"], case["width"], generator=g, device=DEV) * STD).to(TORCH[case["dtype"]]))
    rows = case["out"] * (2 if case["kind"] == "gated" else 1)
    s = dict(x=_activations(g, case["tokens"], case["width"], case["dtype"]))
    s["codes"], s["scales"] = _pack(torch.randn(rows, case["width"], generator=g, device=DEV) * STD)
    s["bias"] = torch.randn(rows, generator=g, device=DEV) * STD
    if case.get("residual"):
        s["residual"] = torch.randn(case["tokens"], case["out"], generator=g, device=DEV) * 4.0
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    return s


def run(s):
    case, x = s["case"], s["x"]
    kind = case["kind"]
    if own:
        from transformers_neuronx_b200.kernels import mxfp4
        if kind == "quantize":
            return mxfp4.dequantize_mxfp4(mxfp4.quantize_mxfp4(x), torch.bfloat16)
        w = mxfp4.Mxfp4Matrix(s["codes"], s["scales"], case["width"])
        a = mxfp4.quantize_mxfp4(x) if kind == "product" or case.get("quantized") else x
        if kind == "gated":
            out = torch.empty((case["tokens"], case["out"]), dtype=x.dtype, device=x.device)
            return mxfp4.gated_gemm_mxfp4(a, w, out, bias=s["bias"], activation=case["act"])
        residual = s.get("residual")
        out = torch.empty((case["tokens"], case["out"]), dtype=x.dtype if residual is None else torch.float32, device=x.device)
        return mxfp4.gemm_mxfp4(a, w, out, bias=s["bias"], residual=residual, activation=case["act"])
    if kind == "quantize":
        return _quantized(x).view(x.shape[0], -1)[:, :x.shape[1]].to(torch.bfloat16)
    a = _quantized(x).view(x.shape[0], -1) if kind == "product" or case.get("quantized") else x.float()
    y = a @ _unpack(s["codes"], s["scales"], case["width"]).T + s["bias"]
    if kind == "gated":
        return (_activation(y[:, :case["out"]], case["act"]) * y[:, case["out"]:]).to(x.dtype)
    y = _activation(y, case["act"])
    return y.to(x.dtype) if "residual" not in s else y + s["residual"]


def work(case):
    if case["kind"] == "quantize":
        n = case["rows"] * case["width"]
        size = 4 if case["dtype"] == "float32" else 2
        return {"bytes": n * size + 2 * n * (1 / 2 + 1 / 32) + 2 * n, "flops": 2 * n}
    t, k, n = case["tokens"], case["width"], case["out"]
    rows = n * (2 if case["kind"] == "gated" else 1)
    out = 8 if case.get("residual") else 2                      # the residual is read and the sum written
    return {"bytes": rows * k * (1 / 2 + 1 / 32) + 2 * t * k + 4 * rows + out * t * n, "flops": 2 * t * rows * k}


# ---- 64 bits -------------------------------------------------------------------------------------------------------
def _exact_quantized(x):
    """The definition in 64 bits, value by value against the eight magnitudes."""
    x = x.double()
    rows, width = x.shape
    x = torch.cat((x, x.new_zeros(rows, -width % 32)), 1).view(rows, -1, 32)
    m = x.abs().amax(-1, keepdim=True)
    e = torch.where(m > 0, torch.ceil(torch.log2(m / 6)), torch.full_like(m, -127.0))
    e = torch.where((m > 6 * torch.exp2(e)), e + 1, torch.where((m > 0) & (m <= 6 * torch.exp2(e - 1)), e - 1, e)).clamp(-127, 127)
    v = x / torch.exp2(e)
    best = torch.zeros_like(v)
    far = v.abs()
    for i, mag in enumerate(MAGNITUDES[1:], 1):
        d = (v.abs() - mag).abs()
        take = (d < far) | ((d == far) & (i % 2 == 0))          # a tie between neighbours goes to the even one
        best, far = torch.where(take, torch.full_like(v, mag), best), torch.where(take, d, far)
    return (torch.where(v < 0, -best, best) * torch.exp2(e)).view(rows, -1)[:, :width]


def _exact_values(codes, scales, width):
    low, high = codes.long() % 16, codes.long() // 16
    c = torch.cat((low.unsqueeze(-1), high.unsqueeze(-1)), -1).flatten(1)
    m = torch.tensor(MAGNITUDES, dtype=torch.float64, device=codes.device)[c % 8] * (1.0 - 2.0 * (c // 8))
    return (m * torch.exp2(scales.double() - 127).repeat_interleave(32, 1))[:, :width]


def exact(case, seed):
    s = _inputs(case, seed)
    x = s["x"].double()
    if case["kind"] == "quantize":
        return _exact_quantized(s["x"])
    if case["kind"] == "product" or case.get("quantized"):
        x = _exact_quantized(s["x"])
    y = torch.matmul(x, _exact_values(s["codes"], s["scales"], case["width"]).t()) + s["bias"].double()
    n = case["out"]
    act = {"none": lambda t: t, "relu": lambda t: t.clamp_min(0), "silu": lambda t: t * torch.sigmoid(t),
           "gelu_new": lambda t: t * torch.sigmoid(1.5957691216057308 * (t + 0.044715 * t ** 3))}[case["act"]]
    if case["kind"] == "gated":
        return act(y[:, :n]) * y[:, n:]
    return act(y) + s["residual"].double() if "residual" in s else act(y)
