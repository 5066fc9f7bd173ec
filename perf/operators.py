"""Microscaled 4-bit numbers: quantisation of rows and linear layers on them, as measurable cases.

A row is cut into blocks of 32 columns (the last one may be shorter).  A block holds one power of two, 2^e with
e = floor(log2(largest magnitude)) - 2, at least -127, and for each column a 4-bit number (sign, two exponent bits, one
mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6), the nearest one to x / 2^e, ties to the even code, 6 beyond 6.  In memory:
codes uint8 [rows, 16 * blocks], the even column in a byte's low half, columns past the last one 0; scales uint8
[rows, blocks], e + 127.

A case is a dict of plain values.  `op` names the operators it runs:

  round_trip   quantise rows, and read the numbers back
  linear       act(x w^T + bias): x bf16, w in 4 bits (weights held small, activations as they come)
  matmul       the same with x quantised in the call: both factors in 4 bits

`swiglu`: the rows of w are interleaved (gate_0, up_0, gate_1, ..) and the result is silu(gate) * up, of out / 2 columns.
`gap`: x is a view of rows that are that many elements longer.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
BLOCK = 32
TYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


# ---- the cases ---------------------------------------------------------------------------------------
def listed():
    return [
        # the hidden state of one decoded token, on its way into a layer on 4-bit numbers
        dict(name="round_trip_token", op="round_trip", rows=1, cols=3584, dtype="bfloat16", gap=0),
        # a weight matrix when a checkpoint is loaded
        dict(name="round_trip_weights", op="round_trip", rows=18944, cols=3584, dtype="bfloat16", gap=0),
        # fp32 rows that end inside a block
        dict(name="round_trip_odd", op="round_trip", rows=1031, cols=4301, dtype="float32", gap=0),
        # one decoded token, a small projection: latency
        dict(name="linear_token_small", op="linear", rows=1, cols=2048, out=2048, bias=False, swiglu=False, gap=0),
        # one decoded token through the gate / up projection
        dict(name="linear_token", op="linear", rows=1, cols=3584, out=37888, bias=False, swiglu=True, gap=0),
        # eight slots of continuous batching through the down projection
        dict(name="linear_slots", op="linear", rows=8, cols=18944, out=3584, bias=False, swiglu=False, gap=0),
        # the prompt of one image and a question through the q | k | v projection
        dict(name="linear_prompt", op="linear", rows=279, cols=3584, out=4608, bias=True, swiglu=False, gap=0),
        # a layer of no round size
        dict(name="linear_odd", op="linear", rows=77, cols=1153, out=1157, bias=True, swiglu=False, gap=0),
        # a prompt portion of the scheduler's step budget through the gate / up projection
        dict(name="linear_portion", op="linear", rows=2048, cols=3584, out=37888, bias=False, swiglu=True, gap=0),
        # 32 slots of continuous batching through the q | k | v projection, both factors in 4 bits
        dict(name="matmul_slots", op="matmul", rows=32, cols=3584, out=4608, bias=True, swiglu=False, gap=0),
        # a prompt portion through the down projection
        dict(name="matmul_portion", op="matmul", rows=2048, cols=18944, out=3584, bias=False, swiglu=False, gap=0),
        # a video of 64 frames through an up projection
        dict(name="matmul_video", op="matmul", rows=16470, cols=3584, out=18944, bias=False, swiglu=False, gap=0),
    ]


def draw(rng):
    def size(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["round_trip", "linear", "linear", "matmul", "matmul"])
    cols = size(64, 18944)
    if rng.random() < 0.6:      # most layers have round widths
        cols = max(64, cols // 64 * 64)
    gap = rng.choice([0, 0, 8, 3])
    if op == "round_trip":
        rows = size(1, 18944)
        return dict(op=op, rows=rows, cols=min(cols, 67000000 // rows), dtype=rng.choice(["bfloat16", "float32"]), gap=gap)
    out = size(64, 37888)
    if rng.random() < 0.6:
        out = max(64, out // 64 * 64)
    rows = size(1, 16470)
    rows = max(1, min(rows, int(1.0e12 / cols / out)))
    swiglu = out % 2 == 0 and rng.random() < 0.3
    return dict(op=op, rows=rows, cols=cols, out=out, bias=rng.random() < 0.5, swiglu=swiglu, gap=gap)


# ---- the plain form ------------------------------------------------------------------------------------
def _quantise(x):
    """fp32 [rows, cols] -> codes, scales"""
    rows, cols = x.shape
    blocks = -(-cols // BLOCK)
    v = torch.nn.functional.pad(x, (0, blocks * BLOCK - cols)).view(rows, blocks, BLOCK)
    top = v.abs().amax(2)
    e = (torch.frexp(top).exponent - 3).clamp(-127, 127)            # frexp's mantissa is in [0.5, 1)
    e = torch.where(top > 0, e, torch.full_like(e, -127))
    v = torch.ldexp(v, -e[..., None])
    a = v.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))      # between neighbours, from 0 on
    q = (torch.round(a / step) * step).clamp(max=6.0)               # half to even: the even code
    table = torch.tensor([0, 1, 2, 3, 4, 4, 5, 5, 6, 6, 6, 6, 7], device=x.device, dtype=torch.uint8)
    c = table[(2 * q).long()] | (torch.signbit(v).to(torch.uint8) << 3)
    c = c.view(rows, blocks * 16, 2)
    return c[..., 0] | (c[..., 1] << 4), (e + 127).to(torch.uint8)


def _values(codes, scales, cols):
    """codes, scales -> fp32 [rows, cols]"""
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], device=codes.device)
    v = table[torch.stack([codes & 15, codes >> 4], 2).long().view(codes.shape[0], -1, BLOCK)]
    return torch.ldexp(v, scales.int()[..., None] - 127).view(codes.shape[0], -1)[:, :cols]


def _finish(z, bias, swiglu):
    if bias is not None:
        z = z + bias.to(z.dtype)
    if swiglu:
        g, u = z[:, 0::2], z[:, 1::2]
        z = g / (1 + torch.exp(-g)) * u
    return z


# ---- inputs ----------------------------------------------------------------------------------------------
def _inputs(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    rows, cols = case["rows"], case["cols"]
    # activations: columns of different size, a few of them far out
    width = torch.exp(0.5 * randn(cols)) * torch.where(torch.rand(cols, generator=g, device=DEV) < 0.005, 20.0, 1.0)
    x = torch.zeros(rows, cols + case["gap"], device=DEV, dtype=TYPES[case.get("dtype", "bfloat16")])
    x[:, :cols] = randn(rows, cols) * width
    s = {"x": x[:, :cols]}
    if case["op"] != "round_trip":
        s["codes"], s["scales"] = _quantise(randn(case["out"], cols) / math.sqrt(cols))
        s["bias"] = (0.1 * randn(case["out"])).to(torch.bfloat16) if case["bias"] else None
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own and case["op"] != "round_trip":
        from vila_b200 import ops
        s["w"] = ops.mx4_pack(s.pop("codes"), s.pop("scales"), case["cols"])   # the layout the products read, made once
    return s


def run(s):
    case, x = s["case"], s["x"]
    if own:
        from vila_b200 import ops
        if case["op"] == "round_trip":
            return ops.mx4_dequantize(ops.mx4_quantize(x), out_dtype=x.dtype)
        if case["op"] == "linear":
            return ops.mx4_linear(x, s["w"], s["bias"], swiglu=case["swiglu"])
        return ops.mx4_matmul(ops.mx4_quantize(x), s["w"], s["bias"], swiglu=case["swiglu"])
    v = x.float()
    if case["op"] != "linear":
        v = _values(*_quantise(v), case["cols"])
    if case["op"] == "round_trip":
        return v.to(x.dtype)
    return _finish(v @ _values(s["codes"], s["scales"], case["cols"]).T, s["bias"], case["swiglu"]).to(x.dtype)


def work(case):
    rows, cols = case["rows"], case["cols"]
    blocks = -(-cols // BLOCK)
    x = rows * cols * (4 if case.get("dtype") == "float32" else 2)
    if case["op"] == "round_trip":      # x read, codes and scales written and read, values written
        return {"bytes": 2 * x + 2 * rows * blocks * 17, "flops": 0}
    out = case["out"]
    written = rows * (out // 2 if case["swiglu"] else out) * 2
    return {"bytes": x + out * blocks * 17 + (2 * out if case["bias"] else 0) + written, "flops": 2 * rows * cols * out}


# ---- the same from the definition, in 64 bits --------------------------------------------------------------
def _nearest64(x):
    """float64 [rows, cols] -> the numbers its microscaled form stands for"""
    rows, cols = x.shape
    pad = -cols % BLOCK
    b = torch.cat([x, x.new_zeros(rows, pad)], 1).reshape(-1, BLOCK)
    top = b.abs().max(1, keepdim=True).values
    e = torch.floor(torch.log2(top.clamp(min=2.0 ** -125)))
    e = torch.where(torch.exp2(e) > top, e - 1, e)      # log2 rounds
    e = torch.where(torch.exp2(e + 1) <= top, e + 1, e)
    unit = torch.exp2(e - 2)
    a = b.abs() / unit
    values = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    got = torch.zeros_like(a)
    for k in range(1, 8):       # past the middle of two neighbours, or on it where the upper one's code is even
        middle = (values[k - 1] + values[k]) / 2
        got = torch.where((a > middle) | ((a == middle) & (k % 2 == 0)), values[k], got)
    return (got * unit * torch.sign(b)).reshape(rows, -1)[:, :cols]


def exact(case, seed):
    s = _inputs(case, seed)
    x = s["x"].double()
    if case["op"] != "linear":
        x = _nearest64(x)
    if case["op"] == "round_trip":
        return x
    codes = torch.stack([s["codes"] % 16, s["codes"] // 16], 2).reshape(case["out"], -1, BLOCK).double()
    sign = torch.where(codes >= 8, -1.0, 1.0).double()
    c = codes % 8
    mag = torch.where(c < 2, c / 2, (1 + (c % 2) / 2) * torch.exp2(torch.floor(c / 2) - 1))
    w = (sign * mag * torch.exp2(s["scales"].double() - 127)[..., None]).reshape(case["out"], -1)[:, : case["cols"]]
    z = x @ w.T
    if s["bias"] is not None:
        z += s["bias"].double()
    if case["swiglu"]:
        gate, up = z[:, 0::2], z[:, 1::2]
        z = gate * torch.sigmoid(gate) * up
    return z
