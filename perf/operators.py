"""The microscaled 4-bit (MXFP4) operators as measured work: quantisation with its way back, dequantisation, the
product of two 4-bit matrices, and the fully connected layer that quantises its activations on the way in.

A block is 32 neighbours along K that share one power-of-two scale (a byte, exponent bias 127); an element is one of
0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign (4 bits, the even element of a pair in the low half of its byte).  Rows are
padded to whole blocks with zeros.  Scale bytes are kept in tiles of 128 rows x 4 blocks (512 bytes, tiles of one
band of rows in K order): byte (row % 32) * 16 + (row % 128 // 32) * 4 + block % 4.

`own = False` computes everything from elementary torch operations; `own = True` makes the package's calls."""
import math

import torch

own = False

BLOCK = 32
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # activations of a small ragged batch on their way into a layer: latency counts
        {"name": "quantize 33x784 f32 rows", "op": "quantize", "rows": 33, "cols": 784, "along": 0, "dtype": "f32"},
        # a prefill's activations, blocks along the features
        {"name": "quantize 8192x8192 bf16 rows", "op": "quantize", "rows": 8192, "cols": 8192, "along": 0, "dtype": "bf16"},
        # a layer's weights stored [in, out]: blocks run down the columns and the result is stored transposed
        {"name": "quantize 4096x11008 f16 columns", "op": "quantize", "rows": 4096, "cols": 11008, "along": 1, "dtype": "f16"},
        # a layer's weights unpacked for a path that wants 16 bits
        {"name": "dequantize 11008x4096 bf16", "op": "dequantize", "rows": 11008, "cols": 4096, "dtype": "bf16"},
        # an odd matrix unpacked for inspection
        {"name": "dequantize 513x1001 f32", "op": "dequantize", "rows": 513, "cols": 1001, "dtype": "f32"},
        # the square product the suite is quoted on
        {"name": "gemm 8192x8192x8192 bf16", "op": "gemm", "M": 8192, "N": 8192, "K": 8192, "dtype": "bf16"},
        # the wide layer of the W8A8 workload
        {"name": "gemm 8192x28672x8192 bf16", "op": "gemm", "M": 8192, "N": 28672, "K": 8192, "dtype": "bf16"},
        # a ragged product whose sums are wanted unrounded (a weight gradient)
        {"name": "gemm 1000x1544x2056 f32", "op": "gemm", "M": 1000, "N": 1544, "K": 2056, "dtype": "f32"},
        # the reference's hidden layer on a ragged batch
        {"name": "gemm 257x512x784 f16", "op": "gemm", "M": 257, "N": 512, "K": 784, "dtype": "f16"},
        # one token through the up projection
        {"name": "linear 1x4096->11008 bf16", "op": "linear", "M": 1, "N": 11008, "K": 4096, "dtype": "bf16", "bias": False, "relu": False},
        # a decode batch through the down projection
        {"name": "linear 16x11008->4096 f16 bias", "op": "linear", "M": 16, "N": 4096, "K": 11008, "dtype": "f16", "bias": True, "relu": False},
        # a prefill through the up projection with its activation
        {"name": "linear 2048x4096->11008 bf16 bias relu", "op": "linear", "M": 2048, "N": 11008, "K": 4096, "dtype": "bf16", "bias": True, "relu": True},
    ]


def _spread(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["quantize", "dequantize", "gemm", "linear"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op in ("quantize", "dequantize"):
        rows = _spread(rng, 1, 16384)
        cols = _spread(rng, 1, min(28672, 8192 * 8192 // rows))
        case = {"op": op, "rows": rows, "cols": cols, "dtype": dtype}
        if op == "quantize":
            case["along"] = rng.choice([0, 1])
        return case
    if op == "gemm":
        case = {"op": op, "M": _spread(rng, 1, 8192), "N": _spread(rng, 8, 28672), "K": _spread(rng, 32, 8192), "dtype": dtype}
        if rng.random() < 0.5:  # half of them in whole blocks of 64, as layers are
            case["N"], case["K"] = -(-case["N"] // 64) * 64, -(-case["K"] // 64) * 64
        return case
    return {"op": op, "M": _spread(rng, 1, 4096), "N": -(-_spread(rng, 8, 11008) // 8) * 8, "K": -(-_spread(rng, 32, 11008) // 8) * 8,
            "dtype": dtype, "bias": rng.random() < 0.5, "relu": rng.random() < 0.5}


# ---------------------------------------------------------------- elementary pieces


def _to_blocks(x):
    """[rows, K] in 32 bits -> [rows, blocks, 32], the last block filled up with zeros."""
    rows, k = x.shape
    pad = -k % BLOCK
    if pad:
        x = torch.cat([x, x.new_zeros(rows, pad)], 1)
    return x.reshape(rows, -1, BLOCK)


def _quantised(x):
    """Block exponents [rows, blocks] and signed element values [rows, blocks, 32] of a matrix in 32 bits."""
    b = _to_blocks(x)
    top = b.abs().amax(-1)
    exponent = torch.where(top > 0, torch.frexp(top)[1] - 3, -127).clamp(-127, 127)  # top = m * 2^e, m in [0.5, 1)
    y = torch.ldexp(b, -exponent.unsqueeze(-1))
    mag = y.abs().clamp(max=6.0)
    step = torch.where(mag < 2, 0.5, torch.where(mag < 4, 1.0, 2.0))
    return exponent, torch.copysign(torch.round(mag / step) * step, y)


def _packed(x):
    """What a user's program holds of a quantised matrix: packed codes and tiled scale bytes."""
    exponent, v = _quantised(x)
    mag = v.abs()
    code = torch.where(mag < 2, mag * 2, torch.where(mag < 4, mag + 2, mag / 2 + 4)).to(torch.uint8)
    code = (code | (torch.signbit(v).to(torch.uint8) << 3)).reshape(x.shape[0], -1)
    q = code[:, 0::2] | (code[:, 1::2] << 4)
    rows, kb = exponent.shape
    bands, tiles = -(-rows // 128), -(-kb // 4)
    s = torch.zeros(bands * 128, tiles * 4, dtype=torch.uint8, device=x.device)
    s[:rows, :kb] = (exponent + 127).to(torch.uint8)
    return q.contiguous(), s.reshape(bands, 4, 32, tiles, 4).permute(0, 3, 2, 1, 4).contiguous()


def _unpacked(q, s):
    """[rows, whole blocks of K] in 32 bits."""
    rows, kb = q.shape[0], q.shape[1] // 16
    code = torch.stack([q & 15, q >> 4], -1).reshape(rows, kb, BLOCK).long()
    table = torch.tensor(GRID + tuple(-g for g in GRID), dtype=torch.float32, device=q.device)
    exponent = s.permute(0, 3, 2, 1, 4).reshape(s.shape[0] * 128, -1)[:rows, :kb].int() - 127
    return torch.ldexp(table[code], exponent.unsqueeze(-1)).reshape(rows, -1)


# ---------------------------------------------------------------- the cases


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(rows, cols):
        """Normal values with a few large ones, as activations have."""
        x = torch.randn(rows, cols, device="cuda", generator=g)
        return x * torch.where(torch.rand(rows, cols, device="cuda", generator=g) < 0.001, 20.0, 1.0)

    def weights(rows, cols):
        return torch.randn(rows, cols, device="cuda", generator=g) * 0.02

    state = dict(case)
    if case["op"] == "quantize":
        state["x"] = normal(case["rows"], case["cols"]).to(DTYPES[case["dtype"]])
    elif case["op"] == "dequantize":
        state["q"], state["s"] = _packed(weights(case["rows"], case["cols"]))
    elif case["op"] == "gemm":
        state["a"], state["sa"] = _packed(normal(case["M"], case["K"]))
        state["b"], state["sb"] = _packed(weights(case["N"], case["K"]))
    else:
        state["x"] = normal(case["M"], case["K"]).to(DTYPES[case["dtype"]])
        state["w"], state["sw"] = _packed(weights(case["N"], case["K"]))
        state["bias"] = torch.randn(case["N"], device="cuda", generator=g) if case["bias"] else None
    return state


def run(state):
    op, dtype = state["op"], DTYPES[state["dtype"]]
    if own:
        import cudaintro_b200 as cb

        if op == "quantize":
            x = state["x"]
            q, s = cb.quantize_mxfp4(x, state["along"])
            return cb.dequantize_mxfp4(q, s, x.shape[1 - state["along"]], dtype)
        if op == "dequantize":
            return cb.dequantize_mxfp4(state["q"], state["s"], state["cols"], dtype)
        if op == "gemm":
            return cb.gemm_mxfp4(state["a"], state["sa"], state["b"], state["sb"], dtype)
        return cb.linear_mxfp4(state["x"], state["w"], state["sw"], state["bias"], relu=state["relu"])
    if op == "quantize":
        x = state["x"].float()
        x = x.t() if state["along"] else x
        exponent, v = _quantised(x)
        return torch.ldexp(v, exponent.unsqueeze(-1)).reshape(x.shape[0], -1)[:, : x.shape[1]].to(dtype).contiguous()
    if op == "dequantize":
        return _unpacked(state["q"], state["s"])[:, : state["cols"]].to(dtype).contiguous()
    if op == "gemm":
        return torch.matmul(_unpacked(state["a"], state["sa"]), _unpacked(state["b"], state["sb"]).t()).to(dtype)
    exponent, v = _quantised(state["x"].float())
    y = torch.matmul(torch.ldexp(v, exponent.unsqueeze(-1)).reshape(state["M"], -1), _unpacked(state["w"], state["sw"]).t())
    if state["bias"] is not None:
        y = y + state["bias"]
    if state["relu"]:
        y = torch.where(y > 0, y, torch.zeros_like(y))
    return y.to(dtype)


def work(case):
    """Inputs once, outputs once; a 4-bit element with its share of a scale is 17/32 of a byte."""
    packed = lambda rows, k: rows * -(-k // BLOCK) * 17  # noqa: E731
    size = SIZE[case["dtype"]]
    if case["op"] == "quantize":  # x in, the packed form out and in again, the values out
        r, c = (case["cols"], case["rows"]) if case["along"] else (case["rows"], case["cols"])
        return {"bytes": 2 * r * c * size + 2 * packed(r, c), "flops": 0}
    if case["op"] == "dequantize":
        return {"bytes": packed(case["rows"], case["cols"]) + case["rows"] * case["cols"] * size, "flops": 0}
    m, n, k = case["M"], case["N"], case["K"]
    a = packed(m, k) if case["op"] == "gemm" else m * k * size
    return {"bytes": a + packed(n, k) + m * n * size + (4 * n if case.get("bias") else 0), "flops": 2 * m * n * k}


# ---------------------------------------------------------------- the definition in 64 bits


def _grid_values_64(x):
    """Values that the format gives a matrix: for each block of 32 the largest power of two not above its largest
    magnitude, over 4, times the nearest element; halfway goes to the element whose code is even."""
    rows, k = x.shape
    below, at = (0.25, 1.25, 2.5, 5.0), (0.75, 1.75, 3.5)  # borders whose middle stays below, and goes up
    table = torch.tensor(GRID, dtype=torch.float64, device=x.device)
    wide = torch.zeros(rows, -(-k // BLOCK) * BLOCK, dtype=torch.float64, device=x.device)
    wide[:, :k] = x
    wide = wide.view(rows, -1, BLOCK)
    top = wide.abs().max(-1, keepdim=True).values
    power = torch.floor(torch.log2(top.clamp(min=2.0**-149)))
    power = power - (torch.exp2(power) > top).double()
    power = power + (torch.exp2(power + 1) <= top).double()
    scale = torch.where(top > 0, torch.exp2((power - 2).clamp(min=-127)), 1.0)
    mag = wide.abs() / scale
    index = sum((mag > b).int() for b in below) + sum((mag >= b).int() for b in at)
    return (torch.sign(wide) * table[index] * scale).reshape(rows, -1)[:, :k].contiguous()


def _values_64(q, s):
    """Element by element from the bits: sign, two bits of exponent, one of mantissa."""
    code = torch.stack((q % 16, q // 16), 2).flatten(1)
    e, m = ((code // 2) % 4).double(), (code % 2).double()
    mag = torch.where(e == 0, m * 0.5, (1 + 0.5 * m) * torch.exp2(e - 1))
    row = torch.arange(code.shape[0], device=q.device).unsqueeze(1)
    k = torch.arange(code.shape[1], device=q.device) // BLOCK
    byte = s.flatten()[((row // 128) * s.shape[1] + k // 4) * 512 + (row % 32) * 16 + (row % 128 // 32) * 4 + k % 4]
    return torch.where(code >= 8, -mag, mag) * torch.exp2(byte.double() - 127)


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "quantize":
        return _grid_values_64(state["x"].t().contiguous() if case["along"] else state["x"])
    if case["op"] == "dequantize":
        return _values_64(state["q"], state["s"])[:, : case["cols"]].contiguous()
    if case["op"] == "gemm":
        return _values_64(state["a"], state["sa"]) @ _values_64(state["b"], state["sb"]).t()
    y = _grid_values_64(state["x"]) @ _values_64(state["w"], state["sw"])[:, : case["K"]].t()
    if case["bias"]:
        y = y + state["bias"].double()
    return y.clamp(min=0) if case["relu"] else y
