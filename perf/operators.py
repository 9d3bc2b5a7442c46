"""Cases and plain forms of the narrow-format Linear operators: the 8-bit activation checkpoints that a training step
keeps for its backward pass, and the microscaled 4-bit (MX, E2M1 with one power-of-two scale per 32 values) quantisation
and products that a frozen network is evaluated with.

Formats, both in blocks of 32 consecutive columns of a row (the last block of a row may be shorter):

  q8   byte = (not x > 0) << 7 | q, value = +-q 2^s; s = e - 6, one more where the largest magnitude's 7-bit rounding
       carries (>= 127.5 / 64 of 2^e), e = floor(log2 max|x|), and s between -127 and 121; q = |x| / 2^s rounded half
       to even, at most 127. The scale byte is s + 127, 255 where the block holds an infinity or NaN (it then reads
       back as NaN).
  mx4  nibble = sign << 3 | index into {0, 0.5, 1, 1.5, 2, 3, 4, 6}, low nibble first; s = floor(log2 max|x|) - 2, not
       below -127; |x| / 2^s rounded to the nearest, half to even, magnitudes over 6 to 6. Scale byte as above.

Code rows are padded to whole blocks, scale rows to a multiple of 4 bytes.
"""
import math
import os
import sys

import torch

own = False

BLOCK = 32
FEAT_ROWS = 203008        # rows of one training step of 8192 rays at 800x800 (8 neighbours per kept sample)
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def listed():
    return [
        # the network's first-layer input (63 positional columns, 128 features, rows of 192 floats) put away in 8 bits
        {"name": "q8 keep feat_net input", "op": "keep", "rows": FEAT_ROWS, "cols": 191, "pad": 1},
        # the same of a handful of rows: what one call costs
        {"name": "q8 keep few rows", "op": "keep", "rows": 37, "cols": 33, "pad": 0},
        # one hidden layer of the neighbour network in a training step, its output kept in 8 bits
        {"name": "q8 forward feat_net layer", "op": "forward", "rows": FEAT_ROWS, "cols": 128, "outs": 128, "pad": 0, "slope": 0.01},
        # a pose network's layer: one row
        {"name": "q8 forward one row", "op": "forward", "rows": 1, "cols": 256, "outs": 256, "pad": 0, "slope": 0.0},
        # the same hidden layer's backward pass from the 8-bit checkpoints
        {"name": "q8 backward feat_net layer", "op": "backward", "rows": FEAT_ROWS, "cols": 128, "outs": 128, "slope": 0.01},
        # the first layer's, for a smaller batch of rays with an odd row count
        {"name": "q8 backward first layer", "op": "backward", "rows": 25601, "cols": 191, "outs": 128, "slope": 0.01},
        # a batch of feature rows into the 4-bit format and back
        {"name": "mx4 quantize feat_net input", "op": "quantize", "rows": FEAT_ROWS, "cols": 191, "pad": 1, "type": "float32"},
        {"name": "mx4 quantize wide half rows", "op": "quantize", "rows": 512, "cols": 4096, "pad": 0, "type": "bfloat16"},
        # one row through a wide layer: the weights' bytes count
        {"name": "mx4 linear one row", "op": "linear", "rows": 1, "cols": 4096, "outs": 4096, "type": "bfloat16", "slope": -1.0},
        # a ragged product
        {"name": "mx4 linear odd", "op": "linear", "rows": 203, "cols": 1000, "outs": 513, "type": "float32", "slope": 0.01},
        # a large one: the matrix units count
        {"name": "mx4 linear large", "op": "linear", "rows": 8192, "cols": 4096, "outs": 4096, "type": "bfloat16", "slope": -1.0},
        # the whole neighbour network (191 -> 128 -> 128 -> 128 -> 128) over a band of a frame, its rows as the gather writes them
        {"name": "mx4 feat_net", "op": "network", "rows": 262144, "cols": 191, "outs": 128, "depth": 4, "pad": 1, "type": "float32",
         "out": "bfloat16", "slope": 0.01},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["keep", "forward", "forward", "backward", "backward", "quantize", "linear", "linear", "network"])
    slope = rng.choice([-1.0, 0.0, 0.01])
    if op in ("keep", "quantize"):
        c = {"op": op, "rows": _log_int(rng, 1, FEAT_ROWS), "cols": _log_int(rng, 1, 512), "pad": rng.choice([0, 1, 5])}
        c["rows"] = min(c["rows"], FEAT_ROWS * 191 // c["cols"])
        if op == "quantize":
            c["type"] = rng.choice(list(DTYPES))
        return c
    if op in ("forward", "backward"):
        c = {"op": op, "rows": _log_int(rng, 1, FEAT_ROWS), "cols": _log_int(rng, 1, 512), "outs": _log_int(rng, 1, 512)}
        c["rows"] = min(c["rows"], FEAT_ROWS * 191 // max(c["cols"], c["outs"]))
        if op == "forward":
            c["pad"] = rng.choice([0, 1, 3])
        return {**c, "slope": slope}
    if op == "network":
        return {"op": op, "rows": _log_int(rng, 64, 262144), "cols": _log_int(rng, 32, 256), "outs": rng.choice([32, 64, 96, 128, 200, 256]),
                "depth": rng.randint(2, 5), "pad": rng.choice([0, 1]), "type": rng.choice(["float32", "bfloat16"]), "out": "bfloat16",
                "slope": rng.choice([0.0, 0.01])}
    return {"op": op, "rows": _log_int(rng, 1, 8192), "cols": _log_int(rng, 32, 4096), "outs": _log_int(rng, 32, 4096),
            "type": rng.choice(list(DTYPES)), "slope": slope}


# --- the formats in plain torch -------------------------------------------------------------------------------------

def _blocks(x):
    """[M, K] as [M, ceil(K / 32), 32] in 32 bits, zeros behind K."""
    M, K = x.shape
    B = -(-K // BLOCK)
    return torch.nn.functional.pad(x.float(), (0, B * BLOCK - K)).reshape(M, B, BLOCK)


def _scale_bytes(amax, carry, shift):
    """Biased exponent of amax (after adding `carry` to its bits) less `shift`, 255 for non-finite amax."""
    byte = (((amax.view(torch.int32) + carry) >> 23) - shift).clamp_(min=0)
    return torch.where(torch.isfinite(amax), byte, torch.full_like(byte, 255))


def _power(byte):
    """2^(byte - 127) in 32 bits, NaN for 255."""
    bits = torch.where(byte == 0, torch.full_like(byte, 0x00400000), byte << 23)
    return torch.where(byte == 255, torch.full_like(byte, 0x7FC00000), bits).view(torch.float32)


def _up(b, byte):
    """b / 2^(byte - 127), exactly (zeros where the block has no scale)."""
    return torch.where((byte == 255)[..., None], torch.zeros_like(b), b) * ((254 - byte.clamp(max=253)) << 23).view(torch.float32)[..., None]


def _q8(x):
    """(code bytes, scale bytes) of x [M, K], as blocks."""
    b = _blocks(x)
    byte = _scale_bytes(_amax(b), 0x10000, 6)
    byte = torch.where(byte == 249, torch.full_like(byte, 248), byte)
    q = torch.round(_up(b.abs(), byte)).clamp_(max=127).to(torch.uint8)
    return torch.where(b > 0, q, q | 0x80), byte


def _q8_values(codes, byte):
    v = (codes & 0x7F).float() * _power(byte)[..., None]
    return torch.where(codes >= 0x80, -v, v)


def _amax(b):
    return torch.where(torch.isfinite(b).all(-1), b.abs().amax(-1), torch.full_like(b[..., 0], math.inf))


def _mx4(x):
    """(code nibbles, one a byte, scale bytes) of x [M, K], as blocks."""
    b = _blocks(x)
    byte = _scale_bytes(_amax(b), 0, 2)
    a = _up(b.abs(), byte)
    # half steps between neighbouring magnitudes; the even index wins a tie
    code = (a > 0.25).to(torch.uint8) + (a >= 0.75).to(torch.uint8) + (a > 1.25).to(torch.uint8) + (a >= 1.75).to(torch.uint8)
    code += (a > 2.5).to(torch.uint8) + (a >= 3.5).to(torch.uint8) + (a > 5.0).to(torch.uint8)
    return code | ((b.view(torch.int32) < 0).to(torch.uint8) << 3), byte


def _mx4_values(codes, byte):
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
    v = table[(codes & 7).long()] * _power(byte)[..., None]
    return torch.where(codes >= 8, -v, v)


def _rows(v, K):
    return v.reshape(v.shape[0], -1)[:, :K]


def _scale_rows(byte):
    return torch.nn.functional.pad(byte, (0, -byte.shape[1] % 4)).to(torch.uint8)


def _mx4_packed(w):
    """(codes [N, 16 B], scales [N, 4 ceil(B / 4)]) of a weight: what a program keeps of it."""
    codes, byte = _mx4(w)
    c = codes.reshape(len(w), -1)
    return c[:, ::2] | (c[:, 1::2] << 4), _scale_rows(byte)


def _mx4_unpacked(codes, scales):
    c = torch.stack([codes & 15, codes >> 4], -1).reshape(len(codes), -1, BLOCK)
    return _mx4_values(c, scales[:, :c.shape[1]].int())


def _act(y, slope):
    return y if slope < 0 else torch.where(y > 0, y, y * slope)


# --- inputs ----------------------------------------------------------------------------------------------------------

def _features(g, M, K, pad, dtype):
    """Rows as the network sees them: positional sines in the first third, features behind, a few rows of zeros."""
    buf = torch.randn(M, K + pad, device="cuda", generator=g)
    third = K // 3
    buf[:, :third] = torch.sin(buf[:, :third] * 40.0)
    buf[:: max(5, M // 7)] *= 0.0 if M > 5 else 1.0
    return buf.to(dtype)[:, :K]


def _weight(g, N, K):
    return (torch.rand(N, K, device="cuda", generator=g) * 2 - 1) * math.sqrt(3.0 / K)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, M, K = case["op"], case["rows"], case["cols"]
    s = {"case": case}
    if op in ("keep", "quantize", "forward", "linear", "network"):
        s["x"] = _features(g, M, K, case.get("pad", 0), DTYPES[case.get("type", "float32")])
    if op in ("keep", "quantize"):
        return s
    N = case["outs"]
    if op == "network":
        s["layers"] = []
        for d in range(case["depth"]):
            w = _weight(g, N, K if d == 0 else N)
            s["layers"].append((*_mx4_packed(w), w.shape[1], 0.1 * torch.randn(N, device="cuda", generator=g)))
        return s
    s["w"], s["b"] = _weight(g, N, K), 0.1 * torch.randn(N, device="cuda", generator=g)
    if op == "linear":
        s["codes"], s["scales"] = _mx4_packed(s.pop("w"))
    if op == "backward":
        s["dy"] = torch.randn(M, N, device="cuda", generator=g) * 1e-4
        for name, v in (("x", _features(g, M, K, 0, torch.float32)), ("y", torch.randn(M, N, device="cuda", generator=g))):
            codes, byte = _q8(v)
            s[name + "_codes"], s[name + "_scales"] = codes.reshape(M, -1), _scale_rows(byte)
    return s


# --- one pass -------------------------------------------------------------------------------------------------------

def _package():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "articulated-point-nerf_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from apn_amd import lowbit
    return lowbit


def _run_own(s):
    lb = _package()
    case = s["case"]
    op, K = case["op"], case["cols"]
    slope = case.get("slope", -1.0)
    slope = None if slope < 0 else slope
    if op == "keep":
        return lb.q8_pack(s["x"]).dequantize(torch.bfloat16)
    if op == "quantize":
        return lb.mx4_quantize(s["x"]).dequantize(torch.bfloat16)
    if op == "forward":
        y, kept = lb.linear_q8(s["x"], s["w"], s["b"], slope)
        return {"y": y, "kept": kept.dequantize(torch.bfloat16)}
    if op == "backward":
        dx, dw, db = lb.linear_q8_backward(s["dy"], s["w"], lb.Q8Rows(s["x_codes"], s["x_scales"], K),
                                           lb.Q8Rows(s["y_codes"], s["y_scales"], case["outs"]), slope)
        return {"dx": dx, "dw": dw, "db": db}
    if op == "linear":
        return lb.mx4_linear(s["x"], lb.MX4Rows(s["codes"], s["scales"], K), s["b"], slope, out_dtype=DTYPES[case["type"]])
    layers = [lb.MX4Layer(lb.MX4Rows(c, sc, k), b, slope) for c, sc, k, b in s["layers"]]
    return lb.mx4_sequential(layers, s["x"], out_dtype=DTYPES[case["out"]])


def run(state):
    if own:
        return _run_own(state)
    s, case = state, state["case"]
    op, K = case["op"], case["cols"]
    slope = case.get("slope", -1.0)
    if op == "keep":
        return _rows(_q8_values(*_q8(s["x"])), K).to(torch.bfloat16)
    if op == "quantize":
        return _rows(_mx4_values(*_mx4(s["x"])), K).to(torch.bfloat16)
    if op == "forward":
        y = _act(torch.matmul(s["x"], s["w"].t()) + s["b"], slope)
        return {"y": y, "kept": _rows(_q8_values(*_q8(y)), case["outs"]).to(torch.bfloat16)}
    if op == "backward":
        M = case["rows"]
        x = _rows(_q8_values(s["x_codes"].reshape(M, -1, BLOCK), s["x_scales"][:, :-(-K // BLOCK)].int()), K)
        dy = s["dy"] if slope < 0 else torch.where(s["y_codes"][:, :case["outs"]] < 0x80, s["dy"], s["dy"] * slope)
        return {"dx": torch.matmul(dy, s["w"]), "dw": torch.matmul(dy.t(), x), "db": dy.sum(0)}
    if op == "linear":
        y = torch.matmul(_rows(_mx4_values(*_mx4(s["x"])), K), _rows(_mx4_unpacked(s["codes"], s["scales"]), K).t())
        return _act(y + s["b"], slope).to(DTYPES[case["type"]])
    h = s["x"]
    for codes, scales, k, b in s["layers"]:
        h = torch.matmul(_rows(_mx4_values(*_mx4(h)), k), _rows(_mx4_unpacked(codes, scales), k).t())
        h = _act(h + b, slope)
    return h.to(DTYPES[case["out"]])


def work(case):
    op, M, K = case["op"], case["rows"], case["cols"]
    N = case.get("outs", 0)
    blocks = lambda k: -(-k // BLOCK)  # noqa: E731
    q8 = lambda k: M * (k + blocks(k))  # noqa: E731
    mx4 = lambda m, k: m * (k / 2 + blocks(k))  # noqa: E731
    size = 4 if case.get("type", "float32") == "float32" else 2
    if op == "keep":
        return {"bytes": 4 * M * K + 2 * q8(K) + 2 * M * K, "flops": 2 * M * K}
    if op == "quantize":
        return {"bytes": size * M * K + 2 * mx4(M, K) + 2 * M * K, "flops": 2 * M * K}
    if op == "forward":   # the checkpoint is written, and read back once into 16 bits
        return {"bytes": 4 * (M * K + N * K + N + M * N) + 2 * q8(N) + 2 * M * N, "flops": 2 * M * N * K}
    if op == "backward":
        return {"bytes": 4 * (M * N + N * K + M * K + N * K + N) + q8(K) + M * N, "flops": 4 * M * N * K}
    if op == "linear":
        return {"bytes": size * (M * K + M * N) + mx4(N, K) + 4 * N, "flops": 2 * M * N * K}
    D = case["depth"]
    return {"bytes": size * M * K + 2 * M * N + mx4(N, K) + (D - 1) * mx4(N, N) + 4 * D * N,
            "flops": 2 * M * N * (K + (D - 1) * N)}


# --- from the definition, in 64 bits --------------------------------------------------------------------------------

def _exact_blocks(x, width):
    """x [M, K] in 64 bits on `width`-bit magnitudes (7: integers; 2: E2M1), read back."""
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for at in range(0, x.shape[1], BLOCK):
        b = x[:, at:at + BLOCK].double()
        top = b.abs().amax(1, keepdim=True)
        part, e = torch.frexp(top)
        e = torch.where(top > 0, e - 1, torch.full_like(e, -1000))
        if width == 7:
            s = (e - 6 + (2 * part >= 127.5 / 64).int()).clamp(min=-127, max=121)
            v = torch.round(torch.ldexp(b, -s)).clamp(-127, 127)
        else:
            s = (e - 2).clamp(min=-127)
            a = torch.ldexp(b, -s).clamp(-6.0, 6.0)
            step = torch.where(a.abs() < 2, 0.5, torch.where(a.abs() < 4, 1.0, 2.0)).double()
            v = torch.round(a / step) * step
        v = torch.ldexp(v, s)
        out[:, at:at + BLOCK] = torch.where(torch.isfinite(b).all(1, keepdim=True), v, torch.full_like(v, math.nan))
    return out


def _exact_kept(codes, scales, K):
    """What 8-bit codes stand for, in 64 bits."""
    low = (codes[:, :K].long() & 127).double() * (1 - 2 * (codes[:, :K].long() >> 7)).double()
    s = scales.long().repeat_interleave(BLOCK, 1)[:, :K] - 127
    return torch.ldexp(low, s)


def _exact_weight(codes, scales, K):
    """What 4-bit codes stand for, in 64 bits: (-1)^sign 2^max(e - 1, 0) (m / 2 + (e > 0)), with e and m the nibble's middle two and last bits."""
    n = torch.empty(len(codes), 2 * codes.shape[1], dtype=torch.int64, device=codes.device)
    n[:, 0::2], n[:, 1::2] = codes.long() % 16, codes.long() // 16
    n = n[:, :K]
    e, m = (n >> 1) & 3, n & 1
    v = torch.ldexp(m / 2.0 + (e > 0).double(), (e - 1).clamp(min=0)) * (1 - 2 * (n >> 3)).double()
    return torch.ldexp(v, scales.long().repeat_interleave(BLOCK, 1)[:, :K] - 127)


def exact(case, seed):
    s = prepare(case, seed)
    op, K = case["op"], case["cols"]
    slope = case.get("slope", -1.0)
    leaky = lambda v: v if slope < 0 else v.clamp(min=0) + slope * v.clamp(max=0)  # noqa: E731
    if op in ("keep", "quantize"):
        return _exact_blocks(s["x"], 7 if op == "keep" else 2)
    if op == "forward":
        y = leaky(torch.addmm(s["b"].double(), s["x"].double(), s["w"].double().t()))
        return {"y": y, "kept": _exact_blocks(y, 7)}
    if op == "backward":
        x = _exact_kept(s["x_codes"], s["x_scales"], K)
        gate = torch.ones((), dtype=torch.float64, device="cuda") if slope < 0 else 1.0 - (1.0 - slope) * (s["y_codes"][:, :case["outs"]] >> 7).double()
        dy = s["dy"].double() * gate
        return {"dx": dy @ s["w"].double(), "dw": (x.t() @ dy).t(), "db": dy.sum(0)}
    if op == "linear":
        y = torch.addmm(s["b"].double(), _exact_blocks(s["x"], 2), _exact_weight(s["codes"], s["scales"], K).t())
        return leaky(y)
    h = s["x"].double()
    for codes, scales, k, b in s["layers"]:
        h = leaky(torch.addmm(b.double(), _exact_blocks(h, 2), _exact_weight(codes, scales, k).t()))
    return h
