"""8-bit floating point rows with a scale per block of 128: quantisation, the norm before a layer, and linear layers, as measurable cases.

A row of activations is cut into blocks of 128 columns (the last one may be shorter), a weight into blocks of 128 rows by 128 columns.  A block
holds one fp32 scale s = max(largest magnitude / 448, 2^-126) and for each element an e4m3 number (sign, four exponent bits, three mantissa
bits, at most 448): the nearest one to x * (1 / s), ties to even; both quotients and the product are rounded to fp32.  A block with an infinity or a NaN
has a NaN for its scale and zeros for its numbers.

A case is a dict of plain values.  `op` names the operator it runs:

  quantize   rows, or (`block_rows` 128) a weight -> numbers and scales
  norm       x += residual (where there is one), then x / sqrt(mean(x^2) + eps) * w -> numbers and scales, and x
  linear     act(a w^T + bias): both factors in 8 bits, fp32 sums, a result in bf16 (`to8`: numbers and scales); `rows` says whether the program
             has a in 8 bits (from a norm or another layer) or as bf16 rows, quantised in the call

`swiglu`: the rows of w are interleaved (gate_0, up_0, gate_1, ..) and the result is silu(gate) * up, of out / 2 columns.
`gap`: x is a view of rows that are that many elements longer.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
BLOCK = 128
TOP = 448.0                 # the largest e4m3 number
EPS = 1e-6
TYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


# ---- the cases ---------------------------------------------------------------------------------------
def listed():
    return [
        # the attention output of one decoded token, on its way into the output projection
        dict(name="quantize_token", op="quantize", rows=1, cols=3584, block_rows=1, dtype="bfloat16", gap=0),
        # the attention output of a video prompt
        dict(name="quantize_video", op="quantize", rows=16470, cols=3584, block_rows=1, dtype="bfloat16", gap=0),
        # a gate / up weight when a checkpoint is loaded
        dict(name="quantize_weight", op="quantize", rows=37888, cols=3584, block_rows=128, dtype="bfloat16", gap=0),
        # the norm before a layer, one decoded token: latency
        dict(name="norm_token", op="norm", rows=1, cols=3584, residual=True, dtype="bfloat16", gap=0),
        # a prompt portion of the scheduler's step budget
        dict(name="norm_portion", op="norm", rows=2048, cols=3584, residual=True, dtype="bfloat16", gap=0),
        # an fp32 residual stream whose rows end inside a block
        dict(name="norm_odd", op="norm", rows=1031, cols=4301, residual=False, dtype="float32", gap=3),
        # one decoded token through the gate / up projection: the weight's bytes
        dict(name="linear_token", op="linear", rows=1, cols=3584, out=37888, bias=False, swiglu=True, to8=False, a="fp8"),
        # eight slots of continuous batching through the down projection
        dict(name="linear_slots", op="linear", rows=8, cols=18944, out=3584, bias=False, swiglu=False, to8=False, a="fp8"),
        # the prompt of one image and a question through the q | k | v projection
        dict(name="linear_prompt", op="linear", rows=279, cols=3584, out=4608, bias=True, swiglu=False, to8=False, a="fp8"),
        # a layer of no round size, rows as they come
        dict(name="linear_odd", op="linear", rows=77, cols=1153, out=1157, bias=True, swiglu=False, to8=False, a="bf16"),
        # a prompt portion through the gate / up projection, its result in 8 bits for the down projection
        dict(name="linear_portion", op="linear", rows=2048, cols=3584, out=37888, bias=False, swiglu=True, to8=True, a="fp8"),
        # a video of 64 frames through the down projection
        dict(name="linear_video", op="linear", rows=16470, cols=18944, out=3584, bias=False, swiglu=False, to8=False, a="fp8"),
    ]


def draw(rng):
    def size(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["quantize", "norm", "linear", "linear", "linear"])
    cols = size(64, 18944)
    if rng.random() < 0.6:      # most layers have round widths
        cols = max(64, cols // 64 * 64)
    if op != "linear":
        rows = size(1, 37888)
        cols = min(cols, max(1, 67000000 // rows))
        case = dict(op=op, rows=rows, cols=cols, dtype=rng.choice(["bfloat16", "float32"]), gap=rng.choice([0, 0, 8, 3]))
        case |= dict(block_rows=rng.choice([1, 1, 128])) if op == "quantize" else dict(residual=rng.random() < 0.6)
        return case
    out = size(64, 37888)
    if rng.random() < 0.6:
        out = max(64, out // 64 * 64)
    rows = size(1, 16470)
    rows = max(1, min(rows, int(1.0e12 / cols / out)))
    swiglu = out % 2 == 0 and rng.random() < 0.3
    return dict(op=op, rows=rows, cols=cols, out=out, bias=rng.random() < 0.5, swiglu=swiglu, to8=rng.random() < 0.3, a=rng.choice(["fp8", "fp8", "bf16"]))


# ---- the plain form ------------------------------------------------------------------------------------
def _blocks(v, block_rows):
    """[rows, cols] -> [row blocks, block_rows, column blocks, 128], zeros past the ends"""
    rows, cols = v.shape
    v = torch.nn.functional.pad(v, (0, -cols % BLOCK, 0, -rows % block_rows))
    return v.view(-1, block_rows, v.shape[1] // BLOCK, BLOCK)


def _quantise(x, block_rows):
    """fp32 [rows, cols] -> numbers (e4m3) and scales"""
    v = _blocks(x, block_rows)
    top = v.abs().amax((1, 3), keepdim=True)
    s = (top / torch.full_like(top, TOP)).clamp(min=2.0 ** -126)       # by a number the GPU's division is a product
    fine = torch.isfinite(top)
    codes = torch.where(fine, v * (1.0 / s), torch.zeros_like(v)).to(torch.float8_e4m3fn)
    s = torch.where(fine, s, torch.full_like(s, math.nan))
    return codes.reshape(-1, v.shape[2] * BLOCK)[: x.shape[0], : x.shape[1]].contiguous(), s[:, 0, :, 0].contiguous()


def _values(codes, scales, block_rows):
    """numbers and scales -> fp32 [rows, cols]"""
    v = _blocks(codes.float(), block_rows) * scales[:, None, :, None]
    return v.reshape(-1, v.shape[2] * BLOCK)[: codes.shape[0], : codes.shape[1]]


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
    if case["op"] == "quantize" and case["block_rows"] > 1:
        wide = torch.zeros(rows, cols + case["gap"], device=DEV, dtype=TYPES[case["dtype"]])
        wide[:, :cols] = randn(rows, cols) / math.sqrt(cols)
        return {"x": wide[:, :cols]}
    # activations: columns of different size, a few of them far out
    width = torch.exp(0.5 * randn(cols)) * torch.where(torch.rand(cols, generator=g, device=DEV) < 0.005, 20.0, 1.0)
    wide = torch.zeros(rows, cols + case.get("gap", 0), device=DEV, dtype=TYPES[case.get("dtype", "bfloat16")])
    wide[:, :cols] = randn(rows, cols) * width
    s = {"x": wide[:, :cols]}
    if case["op"] == "norm":
        s["w"] = (1.0 + 0.2 * randn(cols)).to(torch.bfloat16)
        s["residual"] = randn(rows, cols).to(torch.bfloat16) if case["residual"] else None
    if case["op"] == "linear":
        s["w"] = _quantise(randn(case["out"], cols) / math.sqrt(cols), BLOCK)
        s["bias"] = (0.1 * randn(case["out"])).to(torch.bfloat16) if case["bias"] else None
        if case["a"] == "fp8":
            s["a"] = _quantise(s.pop("x").float(), 1)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own and case["op"] == "linear":
        from vila_b200 import ops
        s["w"] = ops.fp8_pack(*s["w"], block_rows=BLOCK)        # a checkpoint's tensors, taken as they are
        if "a" in s:
            s["a"] = ops.fp8_pack(*s["a"], block_rows=1)        # the form in which a norm or a layer before gives its rows
    return s


def run(s):
    case = s["case"]
    if own:
        from vila_b200 import ops
        if case["op"] == "quantize":
            q = ops.fp8_quantize(s["x"], block_rows=case["block_rows"])
            return {"codes": q.codes, "scales": q.scales}
        if case["op"] == "norm":
            # x stays as it was, so that every pass has the same work: the sum is a tensor of its own
            q, x = ops.fp8_rmsnorm(s["x"], s["w"], EPS, residual=s["residual"])
            return {"codes": q.codes, "scales": q.scales, "x": x}
        y = ops.fp8_linear(s["a"] if case["a"] == "fp8" else s["x"], s["w"], s["bias"], swiglu=case["swiglu"], to8=case["to8"])
        return {"codes": y.codes, "scales": y.scales} if case["to8"] else y
    if case["op"] == "quantize":
        codes, scales = _quantise(s["x"].float(), case["block_rows"])
        return {"codes": codes, "scales": scales}
    if case["op"] == "norm":
        x = s["x"]
        if s["residual"] is not None:
            x = (x.float() + s["residual"].float()).to(x.dtype)
        v = x.float()
        codes, scales = _quantise(v * torch.rsqrt(v.square().mean(1, keepdim=True) + EPS) * s["w"].float(), 1)
        return {"codes": codes, "scales": scales, "x": x}
    a = s["a"] if case["a"] == "fp8" else _quantise(s["x"].float(), 1)
    z = _finish(_values(*a, 1) @ _values(*s["w"], BLOCK).T, s["bias"], case["swiglu"])
    if not case["to8"]:
        return z.to(torch.bfloat16)
    codes, scales = _quantise(z, 1)
    return {"codes": codes, "scales": scales}


def work(case):
    rows, cols = case["rows"], case["cols"]
    blocks = -(-cols // BLOCK)
    size = 4 if case.get("dtype") == "float32" else 2
    if case["op"] == "quantize":
        return {"bytes": rows * cols * (size + 1) + -(-rows // case["block_rows"]) * blocks * 4, "flops": 0}
    if case["op"] == "norm":        # x read; with a residual that read and the sum written
        return {"bytes": rows * cols * (size + 1 + ((2 + size) if case["residual"] else 0)) + cols * 2 + rows * blocks * 4, "flops": 0}
    out = case["out"]
    width = out // 2 if case["swiglu"] else out
    a = rows * (cols + blocks * 4) if case["a"] == "fp8" else rows * cols * 2
    w = out * cols + -(-out // BLOCK) * blocks * 4
    written = rows * (width + -(-width // BLOCK) * 4 if case["to8"] else 2 * width)
    return {"bytes": a + w + (2 * out if case["bias"] else 0) + written, "flops": 2 * rows * cols * out}


# ---- the same from the definition, in 64 bits --------------------------------------------------------------
def _per_element(per_block, block_rows, rows, cols):
    return per_block.repeat_interleave(block_rows, 0)[:rows].repeat_interleave(BLOCK, 1)[:, :cols]


def _nearest64(x, block_rows):
    """float64 [rows, cols] -> the e4m3 numbers and the scales of its 8-bit form"""
    rows, cols = x.shape
    padded = x.new_zeros(rows + -rows % block_rows, cols + -cols % BLOCK)
    padded[:rows, :cols] = x.abs()
    top = torch.stack([b.amax(1) for b in padded.split(BLOCK, 1)], 1)               # [rows, column blocks]
    top = top.view(-1, block_rows, top.shape[1]).amax(1)
    scale = (top / 448).clamp(min=2.0 ** -126).float()                               # a scale is an fp32 number, and so is what
    factor = (1.0 / scale.double()).float().double()                                 # its block is multiplied with
    y = (x * _per_element(factor, block_rows, rows, cols)).float().double()          # so are the products: bf16 numbers meet many ties
    exponent = torch.frexp(y.abs().clamp(min=2.0 ** -6)).exponent - 1                # numbers below 2^-6 are 2^-9 apart
    step = torch.ldexp(torch.ones_like(y), exponent - 3)
    return (torch.round(y / step) * step).clamp(-448, 448), scale.double()


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "quantize":
        codes, scales = _nearest64(s["x"].double(), case["block_rows"])
        return {"codes": codes, "scales": scales}
    if case["op"] == "norm":
        x = s["x"].double()
        if s["residual"] is not None:
            x = x + s["residual"].double()
        stored = x.to(s["x"].dtype).double()        # what is normalised is what the stream holds
        codes, scales = _nearest64(stored / torch.sqrt((stored * stored).mean(1, keepdim=True) + EPS) * s["w"].double(), 1)
        return {"codes": codes, "scales": scales, "x": x}
    if case["a"] == "fp8":
        codes, scales = s["a"][0].double(), s["a"][1].double()
    else:
        codes, scales = _nearest64(s["x"].double(), 1)
    a = codes * _per_element(scales, 1, *codes.shape)
    w = s["w"][0].double() * _per_element(s["w"][1].double(), BLOCK, case["out"], case["cols"])
    z = a @ w.T
    if s["bias"] is not None:
        z += s["bias"].double()
    if case["swiglu"]:
        gate, up = z[:, 0::2], z[:, 1::2]
        z = gate * torch.sigmoid(gate) * up
    if not case["to8"]:
        return z
    codes, scales = _nearest64(z, 1)
    return {"codes": codes, "scales": scales}
