"""Performance cases of the dense feed-forward operators (`zerocool_b200.ffn`): microscaled 4-bit quantisation and products, the gated
block in 16 bits with its gradient.

A microscaled (MX4) matrix [rows, cols] is held as codes, uint8 [rows, cols / 2], two e2m1 values a byte with the even column in the low
half, and scales, one byte e + 127 for 32 columns, laid out in tiles of 128 rows x 4 scales: byte (row % 32) * 16 + (row % 128) / 32 * 4
+ block % 4 of tile (row / 128, block / 4), tiles row-major, 512 bytes each.

A case calls one operator `layers` times with operands of its own each time; `graph` says that the calls are captured once and replayed,
as a serving loop does with short batches. Activations are N(0, 1) with a few channels that are eight times larger, weights N(0, 0.02),
gradients of the block's output N(0, 0.01).
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BASE = dict(op="linear", tokens=1, k=2048, n=2048, dtype="bf16", out="bf16", plain_x=True, layers=1, graph=False)


def case(name, **kw):
    return dict(BASE, name=name, **kw)


def listed():
    return [
        # the activations of a serving batch on their way into a product: latency
        case("quantize_acts_64", op="quantize", tokens=64, k=4096, layers=4, graph=True),
        # a weight matrix from its FP32 master copy: bandwidth
        case("quantize_weight", op="quantize", tokens=8192, k=4096, dtype="fp32"),
        # one user generating: a projection per layer, one token, weights from HBM
        case("linear_1", tokens=1, k=4096, n=8192, layers=8, graph=True),
        # a small batch of generated tokens at hidden 2048, FP32 results
        case("linear_19", tokens=19, k=2048, n=16384, layers=8, graph=True, out="fp32"),
        # an odd head over an odd prompt chunk whose activations are quantised already
        case("linear_257", tokens=257, k=2560, n=10007, plain_x=False),
        # a prompt of 8192 tokens through a square projection
        case("linear_8192", tokens=8192, k=4096, n=8192, plain_x=False),
        # the shared expert of the benchmark's layer, one token
        case("gated4_1", op="gated4", tokens=1, k=2048, n=512, layers=16, graph=True),
        # a wide dense block over a prompt
        case("gated4_4096", op="gated4", tokens=4096, k=4096, n=8192, plain_x=False),
        # the 16-bit block in serving: five tokens
        case("gated_5", op="gated", tokens=5, k=4096, n=8192, layers=2, graph=True),
        # and a prompt chunk of odd length in FP16 at the native shape's hidden size
        case("gated_1001", op="gated", tokens=1001, k=2560, n=8192, dtype="fp16"),
        # a training step of the shared expert alone: short reduction, small weights
        case("step_shared", op="step", tokens=2048, k=2048, n=512),
        # a training step of a wide block
        case("step_wide", op="step", tokens=8191, k=4096, n=8192),
    ]


def draw(rng):
    """One more case: an operator, its sizes spread over their logarithms, types and forms that go with it."""
    def spread(lo, hi, step=1):
        return max(step, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step)

    op = rng.choice(["quantize", "linear", "linear", "gated4", "gated", "step"])
    c = dict(BASE, op=op)
    if op == "quantize":
        c.update(tokens=spread(1, 16384), k=spread(32, 8192, 32), dtype=rng.choice(["bf16", "fp16", "fp32"]))
    elif op in ("linear", "gated4"):
        c.update(tokens=spread(1, 8192), k=spread(64, 8192, 32), n=spread(64, 16384), dtype=rng.choice(["bf16", "fp16", "fp32"]),
                 out=rng.choice(["bf16", "fp16", "fp32"]), plain_x=rng.random() < 0.5)
    else:
        c.update(tokens=spread(1 if op == "gated" else 16, 8192), k=spread(64, 4096, 8), n=spread(64, 8192, 8), dtype=rng.choice(["bf16", "fp16"]))
    if op != "step" and c["tokens"] <= 64:
        c["layers"], c["graph"] = rng.randint(2, 6), True
    most = work(dict(BASE, op="step", tokens=8191, k=4096, n=8192))["flops"]
    while c["layers"] > 1 and c["layers"] * max(1, c["n"]) * c["k"] > 1 << 28:
        c["layers"] -= 1
    while op != "quantize" and work(c)["flops"] > most / 2:
        c["tokens"] = (c["tokens"] + 1) // 2
    return c


def generator(seed, *what):
    g = torch.Generator(device="cuda")
    g.manual_seed((seed * 1000003 + sum((v + 1) * 7919 ** (i + 1) for i, v in enumerate(what))) % (1 << 62))
    return g


def activations(c, seed, layer):
    g = generator(seed, layer, 0)
    x = torch.randn(c["tokens"], c["k"], device="cuda", generator=g)
    x[:, torch.randint(0, c["k"], (max(1, c["k"] // 256),), device="cuda", generator=g)] *= 8
    return x.to(DTYPES[c["dtype"]])


def weight(c, seed, layer, which):
    return torch.randn(c["n"], c["k"], device="cuda", generator=generator(seed, layer, which)) * 0.02


# -- plain forms ---------------------------------------------------------------------------------------------------------------

def exponents(amax):
    """floor(log2 amax) - 2, at least -127 (also of zero and of subnormal values), from the exponent field of an FP32 value."""
    return ((amax.view(torch.int32) >> 23) - 129).clamp(-127, 125)


def tiled(bytes_, cols):
    """Row-major scale bytes [rows, cols / 32] -> the tile layout (what is left over is 0)."""
    rows, blocks = bytes_.shape
    full = torch.zeros(-(-rows // 128) * 128, -(-blocks // 4) * 4, dtype=torch.uint8, device=bytes_.device)
    full[:rows, :blocks] = bytes_
    return full.view(-1, 4, 32, full.shape[1] // 4, 4).permute(0, 3, 2, 1, 4).contiguous().view(-1)


def untiled(scales, rows, cols):
    tiles = -(-cols // 128)
    return scales.view(-1, tiles, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(-1, tiles * 4)[:rows, :cols // 32]


def plain_quantize(x):
    """-> codes, scales of a finite matrix."""
    rows, cols = x.shape
    b = x.float().view(rows, cols // 32, 32)
    e = exponents(b.abs().amax(2))
    v = torch.ldexp(b.double(), -e.unsqueeze(2))
    a = v.abs()
    # thresholds half-way between 0, .5, 1, 1.5, 2, 3, 4, 6; a tie goes to the code with the even last bit
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)) + 8 * torch.signbit(v).to(torch.uint8)
    code = code.to(torch.uint8).view(rows, cols // 2, 2)
    return code[:, :, 0] | code[:, :, 1] << 4, tiled((e + 127).to(torch.uint8), cols)


def plain_dequantize(codes, scales):
    rows, cols = codes.shape[0], codes.shape[1] * 2
    c = torch.stack((codes & 15, codes >> 4), 2)
    m = c & 7                                       # 0, 1/2, then (2 + last bit) 2^(m / 2 - 2)
    v = torch.where(m < 2, m * 0.5, torch.ldexp(2.0 + (m & 1), (m >> 1).float() - 2))
    v = torch.where(c > 7, -v, v).view(rows, cols // 32, 32)
    return (v * torch.exp2(untiled(scales, rows, cols).float() - 127).unsqueeze(2)).view(rows, cols)


def plain_x(c, o):
    return plain_dequantize(*(plain_quantize(o["x"]) if c["plain_x"] else o["xq"]))


def silu(v):
    return v / (1 + torch.exp(-v))


def plain(c, o):
    if c["op"] == "quantize":
        return plain_dequantize(*plain_quantize(o["x"])).to(torch.bfloat16)
    if c["op"] == "linear":
        return (plain_x(c, o) @ plain_dequantize(*o["w"][0]).T).to(DTYPES[c["out"]])
    if c["op"] == "gated4":
        x = plain_x(c, o)
        return (silu(x @ plain_dequantize(*o["w"][0]).T) * (x @ plain_dequantize(*o["w"][1]).T)).to(DTYPES[c["out"]])
    t, x, (gate, up) = DTYPES[c["dtype"]], o["x"].float(), (w.float() for w in o["w"])
    g, u = x @ gate.T, x @ up.T
    h = (silu(g) * u).to(t)
    if c["op"] == "gated":
        return h
    s, dh = torch.sigmoid(g), o["dh"].float()
    dg, du = dh * u * s * (1 + g * (1 - s)), dh * g * s
    return {"h": h, "dx": (dg @ gate + du @ up).to(t), "dgate": (dg.T @ x).to(t), "dup": (du.T @ x).to(t)}


# -- the framework's operators -------------------------------------------------------------------------------------------------

def called(c, o):
    from zerocool_b200 import ffn
    if c["op"] == "quantize":
        return ffn.mx4_dequantize(ffn.mx4_quantize(o["x"]), torch.bfloat16)
    if c["op"] in ("linear", "gated4"):
        x = o["x"] if c["plain_x"] else ffn.Mx4(*o["xq"])
        w = [ffn.Mx4(*q) for q in o["w"]]
        return (ffn.mx4_linear if c["op"] == "linear" else ffn.mx4_gated)(x, *w, out_dtype=DTYPES[c["out"]])
    if c["op"] == "gated":
        return ffn.gated_forward(o["x"], *o["w"])
    h, g, u = ffn.gated_forward(o["x"], *o["w"], save=True)
    dx, dgate, dup = ffn.gated_backward(o["dh"], o["x"], *o["w"], g, u)
    return {"h": h, "dx": dx, "dgate": dgate, "dup": dup}


def operands(c, seed, layer):
    o = {"x": activations(c, seed, layer)}
    if c["op"] == "quantize":
        return o
    o["w"] = [weight(c, seed, layer, 1 + i) for i in range(1 if c["op"] == "linear" else 2)]
    if c["op"] in ("linear", "gated4"):
        o["w"] = [plain_quantize(w) for w in o["w"]]
        if not c["plain_x"]:
            o["xq"] = plain_quantize(o.pop("x"))
        return o
    o["w"] = [w.to(DTYPES[c["dtype"]]) for w in o["w"]]
    if c["op"] == "step":
        o["dh"] = (torch.randn(c["tokens"], c["n"], device="cuda", generator=generator(seed, layer, 9)) * 0.01).to(DTYPES[c["dtype"]])
    return o


def calls(state):
    form = called if own else plain
    return [form(state["case"], o) for o in state["operands"]]


def prepare(case, seed):
    state = {"case": case, "operands": [operands(case, seed, layer) for layer in range(case["layers"])]}
    if case["graph"]:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            calls(state)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            state["outs"] = calls(state)
        state["graph"] = graph
    return state


def run(state):
    if "graph" in state:
        state["graph"].replay()
        return state["outs"]
    return calls(state)


def work(case):
    c = case
    T, K, N = c["tokens"], c["k"], c["n"]
    e = 4 if c["dtype"] == "fp32" else 2
    mx = 17 / 32                                    # bytes of a microscaled value
    if c["op"] == "quantize":                       # to codes, and back to BF16 values
        return {"bytes": c["layers"] * T * K * (e + 2 * mx + 2), "flops": 0}
    if c["op"] in ("linear", "gated4"):
        mats = 1 if c["op"] == "linear" else 2
        rows = T * K * (e if c["plain_x"] else mx) + T * N * (4 if c["out"] == "fp32" else 2)
        return {"bytes": c["layers"] * (mats * N * K * mx + rows), "flops": c["layers"] * 2.0 * mats * T * N * K}
    if c["op"] == "gated":
        return {"bytes": c["layers"] * 2 * (2 * N * K + T * K + T * N), "flops": c["layers"] * 4.0 * T * N * K}
    # forward and backward: x, dh, both weights in; h, dx and both gradients out
    return {"bytes": c["layers"] * 2 * (4 * N * K + 2 * T * K + 2 * T * N), "flops": c["layers"] * 12.0 * T * N * K}


# -- 64 bits, from the definitions ---------------------------------------------------------------------------------------------

def values64(codes, scales):
    """Values of a microscaled matrix, its scale bytes found by their index in the tile layout."""
    rows, cols = codes.shape[0], codes.shape[1] * 2
    nibble = torch.empty(rows, cols, dtype=torch.long, device=codes.device)
    nibble[:, 0::2], nibble[:, 1::2] = codes.long() & 15, codes.long() >> 4
    expo, last = (nibble >> 1) & 3, nibble & 1
    size = torch.where(expo == 0, 0.5 * last.double(), (1 + 0.5 * last.double()) * 2.0 ** (expo - 1).double())
    r, b = torch.arange(rows, device=codes.device)[:, None], torch.arange(cols // 32, device=codes.device)[None, :]
    at = (r // 128 * -(-cols // 128) + b // 4) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + b % 4
    scale = 2.0 ** (scales[at].double() - 127)
    return torch.where(nibble >= 8, -size, size) * scale.repeat_interleave(32, dim=1)


def rounded64(x):
    """x rounded to microscaled values, in 64 bits: the exponent by frexp, the e2m1 grid by rounding to multiples of its spacing."""
    rows, cols = x.shape
    b = x.double().view(rows, -1, 32)
    top = b.abs().amax(2, keepdim=True)
    e = (torch.frexp(top).exponent - 3).clamp(-127, 125)
    e = torch.where(top == 0, torch.full_like(e, -127), e)
    v = b * 2.0 ** -e.double()
    step = torch.where(v.abs() < 2, 0.5, torch.where(v.abs() < 4, 1.0, 2.0))
    return ((torch.round(v / step) * step).clamp(-6, 6) * 2.0 ** e.double()).view(rows, cols)


def exact(case, seed):
    c, outs = case, []
    for layer in range(c["layers"]):
        o = operands(c, seed, layer)
        if c["op"] == "quantize":
            outs.append(rounded64(o["x"]))
            continue
        if c["op"] in ("linear", "gated4"):
            x = rounded64(o["x"]) if c["plain_x"] else values64(*o["xq"])
            y = [x @ values64(*q).T for q in o["w"]]
            outs.append(y[0] if c["op"] == "linear" else y[0] * torch.sigmoid(y[0]) * y[1])
            continue
        x, gate, up = o["x"].double(), o["w"][0].double(), o["w"][1].double()
        g, u = x @ gate.T, x @ up.T
        s = torch.sigmoid(g)
        if c["op"] == "gated":
            outs.append(g * s * u)
            continue
        dh = o["dh"].double()
        dg, du = dh * u * (s + g * s * (1 - s)), dh * g * s
        outs.append({"h": g * s * u, "dx": dg @ gate + du @ up, "dgate": dg.T @ x, "dup": du.T @ x})
    return outs
