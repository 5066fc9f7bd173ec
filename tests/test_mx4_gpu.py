"""GPU: microscaled 4-bit rows against their restatement in float64."""
import math

import pytest
import torch

from tests import mx4_reference as R

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def rand(seed, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


# ---- quantisation: bit by bit -------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("rows, cols", [(1, 1), (1, 31), (1, 32), (3, 33), (2, 255), (129, 256), (5, 257), (130, 1000), (7, 3584)])
def test_quantise_is_the_definition(cuda, rows, cols, dtype):
    from vila_b200 import ops
    x = (rand(1, rows, cols) * torch.exp(2 * rand(2, 1, cols))).to(dtype)
    codes, scales = R.quantise(x)
    q = ops.mx4_quantize(x.to(cuda))
    assert q.shape == (rows, cols)
    assert torch.equal(q.codes.cpu(), codes)
    assert torch.equal(q.scales.cpu(), R.tiled(scales, cols))       # padding rows and blocks are 0
    got_codes, got_scales = ops.mx4_unpack(q)
    assert torch.equal(got_codes.cpu(), codes) and torch.equal(got_scales.cpu(), scales)
    want = R.values(codes, scales, cols)
    assert torch.equal(ops.mx4_dequantize(q, out_dtype=torch.float32).cpu().double(), want)
    assert torch.equal(ops.mx4_dequantize(q).cpu().double(), want)  # a 4-bit number times a power of two is a bf16 number


def test_quantise_edges(cuda):
    from vila_b200 import ops
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.999, -0.25, -0.75, -5.0, 6.0, 4.0, -0.0, 0.0, 0.125])
    x = torch.zeros(12, 64)
    x[0, :16] = ties
    x[1, :16] = ties * 2.0 ** 100
    x[2, :16] = ties * 2.0 ** -120
    x[3, :4] = torch.tensor([2.0 ** -149, 2.0 ** -140, 0.0, -(2.0 ** -130)])        # fp32 subnormals
    x[4, 32:36] = torch.tensor([3.4028234e38, -3.4028234e38, 1e38, 1.0])
    x[5, 3] = math.inf
    x[6, 40] = math.nan
    x[7, 3], x[7, 4] = math.nan, -math.inf
    x[8] = 6.0
    x[9, 0] = 2.0 ** -126
    x[10, 0] = 2.0 ** -125
    x[11] = -1e-45
    codes, scales = R.quantise(x)
    q = ops.mx4_quantize(x.to(cuda))
    got_codes, got_scales = ops.mx4_unpack(q)
    assert torch.equal(got_scales.cpu(), scales)
    assert torch.equal(got_codes.cpu(), codes)
    back = ops.mx4_dequantize(q, out_dtype=torch.float32).cpu()
    want = R.values(codes, scales, 64).float()
    assert torch.equal(torch.isnan(back), torch.isnan(want)) and torch.equal(back.nan_to_num(7.0), want.nan_to_num(7.0))
    assert torch.isnan(back[5, :32]).all() and not torch.isnan(back[5, 32:]).any()


@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("gap, off", [(8, 0), (3, 0), (8, 1), (0, 3)])
def test_quantise_views(cuda, gap, off, dtype):
    from vila_b200 import ops
    wide = rand(3, 70, 300 + gap + off).to(dtype)
    x = wide[:, off:off + 300]
    codes, scales = R.quantise(x)
    q = ops.mx4_quantize(wide.to(cuda)[:, off:off + 300])
    assert torch.equal(q.codes.cpu(), codes) and torch.equal(q.scales.cpu(), R.tiled(scales, 300))


def test_quantise_broadcast_rows_no_rows_and_pack(cuda):
    from vila_b200 import ops
    x = rand(4, 1, 96).to(cuda)
    q = ops.mx4_quantize(x.expand(5, 96))
    one = R.quantise(x.cpu())
    assert torch.equal(q.codes.cpu(), one[0].expand(5, -1)) and torch.equal(ops.mx4_unpack(q)[1].cpu(), one[1].expand(5, -1))
    none = ops.mx4_quantize(torch.empty(0, 96, device=cuda))
    assert none.shape == (0, 96) and ops.mx4_dequantize(none).shape == (0, 96)
    # plain codes and scales; columns past the last one come with something in them
    codes, scales = R.quantise(rand(5, 9, 41))
    dirty = codes.clone()
    dirty[:, 20] |= 0x70
    dirty[:, 21:] = 0x55
    kept = dirty.to(cuda)
    p = ops.mx4_pack(kept, scales.to(cuda), 41)
    assert torch.equal(p.codes.cpu(), codes) and torch.equal(p.scales.cpu(), R.tiled(scales, 41))
    assert torch.equal(kept.cpu(), dirty)
    assert torch.equal(ops.mx4_dequantize(p, out_dtype=torch.float32).cpu().double(), R.values(codes, scales, 41))


# ---- products --------------------------------------------------------------------------------------------
def act64(z, name, pair=None):
    if name == "none":
        return z
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "relu2":
        return z.clamp(min=0) ** 2
    if name == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    if name == "gelu_erf":
        return 0.5 * z * (1 + torch.erf(z / math.sqrt(2)))
    if name == "xielu":     # act_params (0.7, 0.4)
        return torch.where(z > 0, 0.7 * z * z + z / 2, 0.4 * (torch.exp(z.clamp(max=0)) - 1 - z) + z / 2)
    g, u = z[:, 0::2], z[:, 1::2]
    if name == "swiglu":
        return g * torch.sigmoid(g) * u
    if name == "geglu":
        return act64(g, "gelu_tanh") * u
    g, u = g.clamp(max=2.0), u.clamp(-2.0, 2.0)     # glu_clamp (1.5, 2.0)
    return g * torch.sigmoid(1.5 * g) * (u + 1)


def act_args(name):
    from vila_b200 import ops
    return {"none": {}, "silu": dict(act=ops.ACT_SILU), "relu2": dict(act=ops.ACT_RELU2), "gelu_tanh": dict(act=ops.ACT_GELU_TANH),
            "gelu_erf": dict(act=ops.ACT_GELU_ERF), "xielu": dict(act=ops.ACT_XIELU, act_params=(0.7, 0.4)), "swiglu": dict(swiglu=True),
            "geglu": dict(geglu=True), "glu_clamp": dict(glu_clamp=(1.5, 2.0))}[name]


def check_product(got, x, w, bias, act="none"):
    """got (bf16) against act(x w^T + bias) in float64, element by element.  Sums: a tensor-core step of 16 products truncates by
    at most 2^-22 of the sum of magnitudes S, so does the fp32 addition behind it; with K / 16 + 8 steps dz = S (K / 16 + 8) 2^-22.
    The activations' derivatives are at most 1.13 but for the squares (2 |z| a) and the gates (the other factor): dz enters
    through the corners z +- dz, twice.  fp32 evaluation of the activation: 2^-20 relative; and 1 + tanh, 1 + erf and u + 1 lose up to
    2^-22 (tanhf and erff are within 2 units of 2^-24 of a value near -1, the addition rounds once more), which the other factor,
    z / 2 or the gate, multiplies.  Last, the rounding to bf16: 2^-8 relative."""
    x, w = x.double().cpu(), w.double().cpu()
    z, S = x @ w.T, x.abs() @ w.abs().T
    if bias is not None:
        z, S = z + bias.double().cpu(), S + bias.double().cpu().abs()
    dz = S * ((x.shape[1] / 16 + 8) * 2.0 ** -22)
    want = act64(z, act)
    off = torch.zeros_like(want)
    even = torch.zeros_like(dz)
    even[:, 0::2] = dz[:, 0::2]
    for a in (1, -1):
        for b in (1, -1):
            off = torch.maximum(off, (act64(z + a * even + b * (dz - even), act) - want).abs())
    cancelled = torch.zeros_like(want)
    if act in ("gelu_tanh", "gelu_erf"):
        cancelled = z.abs() * 2.0 ** -22
    elif act in ("geglu", "glu_clamp"):
        cancelled = z[:, 0::2].abs() * (z[:, 1::2].abs() + 1) * 2.0 ** -22
    bound = 2 * off + cancelled + want.abs() * (2.0 ** -8 + 2.0 ** -20) + 2.0 ** -133
    err = (got.double().cpu() - want).abs()
    assert got.dtype == BF and err.shape == bound.shape
    assert (err <= bound).all(), (err / bound).max().item()


def weight(seed, n, k, cuda, spread=0.0):
    from vila_b200 import ops
    w = rand(seed, n, k) / math.sqrt(k) * torch.exp(spread * rand(seed + 1, n, 1))
    codes, scales = R.quantise(w)
    return ops.mx4_pack(codes.to(cuda), scales.to(cuda), k), R.values(codes, scales, k)


SIZES = [(1, 2, 32), (1, 128, 64), (1, 300, 2048), (3, 129, 95), (7, 64, 1153), (8, 1000, 512), (9, 130, 4000), (16, 256, 1024),
         (17, 384, 300), (33, 128, 640), (64, 514, 1000), (65, 1157, 1153), (100, 640, 256), (129, 300, 2080), (200, 130, 96), (300, 770, 520),
         (520, 258, 1056), (2600, 2570, 800)]


# more tiles than rows cut into 4-bit rows are used for: unpacked weights, by tile size (64, 96, 128 rows, pairs), rows off 16-byte
# boundaries (odd K), K of one step, of half a stage, several rounds of the rings, several tiles a CTA
UNPACKED = [(20, 16000, 96), (60, 12000, 520), (33, 9700, 1153), (90, 12000, 520), (96, 6300, 32), (120, 12000, 776), (200, 20000, 300),
            (1200, 5000, 520), (700, 5001, 577), (1031, 2500, 1600)]


@pytest.mark.parametrize("M, N, K", SIZES + UNPACKED)
def test_linear(cuda, M, N, K):
    from vila_b200 import ops
    q, w = weight(M, N, K, cuda, spread=1.0)
    x = (rand(7, M, K) * torch.exp(rand(8, 1, K))).to(BF)
    bias = rand(9, N).to(BF)
    check_product(ops.mx4_linear(x.to(cuda), q), x, w, None)
    check_product(ops.mx4_linear(x.to(cuda), q, bias.to(cuda)), x, w, bias)


@pytest.mark.parametrize("M, N, K", SIZES)
def test_matmul(cuda, M, N, K):
    from vila_b200 import ops
    q, w = weight(M, N, K, cuda, spread=1.0)
    x = (rand(7, M, K) * torch.exp(rand(8, 1, K))).to(BF)
    a = ops.mx4_quantize(x.to(cuda))
    codes, scales = R.quantise(x)
    bias = rand(9, N).to(BF)
    check_product(ops.mx4_matmul(a, q), R.values(codes, scales, K), w, None)
    check_product(ops.mx4_matmul(a, q, bias.to(cuda)), R.values(codes, scales, K), w, bias)


@pytest.mark.parametrize("M", [1, 12, 70, 300])
@pytest.mark.parametrize("act", ["silu", "relu2", "gelu_tanh", "gelu_erf", "xielu", "swiglu", "geglu", "glu_clamp"])
@pytest.mark.parametrize("four", [False, True])
def test_activations(cuda, M, act, four):
    from vila_b200 import ops
    q, w = weight(20, 258, 320, cuda)
    x, bias = (2 * rand(21, M, 320)).to(BF), rand(22, 258).to(BF)
    if four:
        got = ops.mx4_matmul(ops.mx4_quantize(x.to(cuda)), q, bias.to(cuda), **act_args(act))
        x = R.values(*R.quantise(x), 320)
    else:
        got = ops.mx4_linear(x.to(cuda), q, bias.to(cuda), **act_args(act))
    check_product(got, x, w, bias, act)


def test_few_rows_of_a_wide_layer(cuda):
    """rows cut into 4-bit rows: several tiles of tokens (16 rows) and K over a cluster"""
    from vila_b200 import ops
    for M, N, K in ((1, 20000, 1000), (3, 9000, 2080), (8, 5000, 4000), (16, 6000, 3000), (2, 384, 50000)):
        q, w = weight(M, N, K, cuda)
        x, bias = rand(7, M, K).to(BF), rand(9, N).to(BF)
        check_product(ops.mx4_linear(x.to(cuda), q, bias.to(cuda)), x, w, bias)


@pytest.mark.parametrize("act", ["silu", "relu2", "gelu_tanh", "gelu_erf", "xielu", "swiglu", "geglu", "glu_clamp"])
@pytest.mark.parametrize("M, N", [(1, 60002), (60, 9002), (90, 9002), (120, 9002), (700, 5002)])
def test_activations_of_wide_layers(cuda, M, N, act):
    from vila_b200 import ops
    q, w = weight(20, N, 320, cuda)
    x, bias = (2 * rand(21, M, 320)).to(BF), rand(22, N).to(BF)
    check_product(ops.mx4_linear(x.to(cuda), q, bias.to(cuda), **act_args(act)), x, w, bias, act)


@pytest.mark.parametrize("M, N", [(2, 200), (40, 200), (300, 200), (2, 70000), (60, 9000), (700, 5000)])
@pytest.mark.parametrize("gap, off", [(8, 0), (3, 0), (8, 1), (0, 2)])
def test_views(cuda, M, N, gap, off):
    from vila_b200 import ops
    q, w = weight(30, N, 288, cuda)
    wide = rand(31, M, 288 + gap + off).to(BF)
    out = torch.full((M, N + 11), 7.0, dtype=BF, device=cuda)
    got = ops.mx4_linear(wide.to(cuda)[:, off:off + 288], q, out=out[:, 5:5 + N])
    assert got.data_ptr() == out[:, 5:].data_ptr()
    check_product(got, wide[:, off:off + 288], w, None)
    assert (out[:, :5] == 7).all() and (out[:, 5 + N:] == 7).all()


@pytest.mark.parametrize("N, K, four", [(200, 288, False), (70000, 288, False), (200, 288, True)])
def test_one_row_of_any_stride(cuda, N, K, four):
    """a single row, whose stride means nothing, as it comes out of a transposed column"""
    from vila_b200 import ops
    q, w = weight(34, N, K, cuda)
    x, out = torch.empty(K, 1, dtype=BF, device=cuda).T, torch.full((N, 1), 7.0, dtype=BF, device=cuda)
    row = rand(35, 1, K).to(BF)
    x.copy_(row)
    assert x.stride(0) == 1 and out.T.stride(0) == 1
    if four:
        ops.mx4_matmul(ops.mx4_quantize(x), q, out=out.T)
        row = R.values(*R.quantise(row), K)
    else:
        ops.mx4_linear(x, q, out=out.T)
    check_product(out.T, row, w, None)


@pytest.mark.parametrize("M, N", [(3, 200), (40, 200), (3, 70000), (60, 9000), (700, 5000)])
def test_broadcast_rows(cuda, M, N):
    from vila_b200 import ops
    q, w = weight(32, N, 288, cuda)
    x = rand(33, 1, 288).to(BF)
    got = ops.mx4_linear(x.to(cuda).expand(M, 288), q)
    check_product(got, x.expand(M, 288), w, None)
    assert (got == got[:1]).all()


@pytest.mark.parametrize("M, N, four", [(M, 140, four) for M in (1, 8, 16, 50, 300) for four in (False, True)] +
                         [(2, 40000, False), (60, 9000, False), (90, 9000, False), (700, 5000, False)])
def test_scales_over_the_whole_range(cuda, M, N, four):
    """blocks of one row whose sizes are 2^40 apart, rows that differ by 2^60"""
    from vila_b200 import ops
    K = 512
    sizes = torch.tensor([2.0 ** -20, 2.0 ** 20, 1.0, 2.0 ** -5]).repeat_interleave(32).repeat(K // 128)
    rows = torch.exp2(torch.arange(N).float() % 61 - 30)
    codes, scales = R.quantise(rand(40, N, K) * sizes * rows[:, None])
    x = (rand(41, M, K) / sizes * torch.exp2(torch.arange(M).float() % 41 - 20)[:, None]).to(BF)
    q, w = ops.mx4_pack(codes.to(cuda), scales.to(cuda), K), R.values(codes, scales, K)
    if four:
        check_product(ops.mx4_matmul(ops.mx4_quantize(x.to(cuda)), q), R.values(*R.quantise(x), K), w, None)
    else:
        check_product(ops.mx4_linear(x.to(cuda), q), x, w, None)


def ends_of_the_range(M, N, cuda, four, top=118):
    """Rows and weights whose blocks' scales lie at the ends of the range, each block of rows against one of weights that brings the
    products near 1 if there is one, else as near as 2^top allows.  Block 3 of the weights is zeros under the largest
    scale, block 7 numbers of the least size under it.  -> what the product takes, and float64 values of both"""
    from vila_b200 import ops
    K = 512
    base = torch.tensor([0, 1, 2, 254, 30, 127, 200, 254, 240, 250, 252, 13, 64, 190, 252, 0])
    codes, scales = R.quantise(rand(40, N, K))
    scales = (base + (torch.arange(N)[:, None] % 3 - 1) * ((base > 3) & (base < 251))).to(torch.uint8)
    codes[:, 3 * 16:4 * 16] = 0
    codes[:, 7 * 16:8 * 16] &= 0x99      # +-0, +-0.5: what 2^127 leaves in fp32's range
    e = (127 - base).clamp(-125, top).double()
    x = (rand(41, M, K).double() * torch.exp2(e).repeat_interleave(32) * torch.exp2(torch.arange(M).double() % 2)[:, None]).to(BF)
    q, w = ops.mx4_pack(codes.to(cuda), scales.to(cuda), K), R.values(codes, scales, K)
    if not four:
        return x.to(cuda), q, x, w
    a_codes, a_scales = R.quantise(x)
    a_codes[:, 5 * 16:6 * 16] = 0
    a_scales[:, 5] = 254                 # zeros under the largest scale again
    return ops.mx4_pack(a_codes.to(cuda), a_scales.to(cuda), K), q, R.values(a_codes, a_scales, K), w


@pytest.mark.parametrize("top", [118, 60])
@pytest.mark.parametrize("M, N, four", [(1, 200, False), (3, 200, False), (8, 2000, False), (3, 70000, False), (12, 300, False), (40, 200, False),
                                        (60, 9000, False), (90, 9000, False), (120, 9000, False), (700, 5000, False), (3, 200, True), (40, 200, True), (100, 200, True), (300, 200, True), (700, 500, True)])
def test_scales_at_the_ends_of_their_range(cuda, M, N, four, top):
    """The bound is check_product's: a tensor-core step, an addition, and a rounding to bf16 whose least step is 2^-133; scales are powers
    of two, and add nothing to it as long as no intermediate result leaves fp32's range."""
    from vila_b200 import ops
    x, q, x64, w = ends_of_the_range(M, N, cuda, four, top)
    got = ops.mx4_matmul(x, q) if four else ops.mx4_linear(x, q)
    check_product(got, x64, w, None)


@pytest.mark.parametrize("M, N, K", [(3, 150, 416), (3, 50000, 416), (12, 150, 416), (12, 300, 8200), (40, 150, 416), (60, 9000, 416), (700, 5000, 416)])
def test_small_entries_of_rows(cuda, M, N, K):
    """Every kernel reads small entries to their last bit: rows of 2^-100 down to bf16's least step 2^-133, on weights of 2^90, and rows that hold
    entries at both ends.  A block's largest entry leaves 2^-31 of itself (see test_infinities_and_sums_beyond_the_range)."""
    from vila_b200 import ops
    codes, scales = R.quantise(rand(50, N, K))
    scales = scales + 90
    q, w = ops.mx4_pack(codes.to(cuda), scales.to(cuda), K), R.values(codes, scales, K)
    x = (rand(51, M, K).double() * torch.exp2(-100 - 3.0 * (torch.arange(M) % 13).double())[:, None]).to(BF)
    x[1] = (torch.exp2(-133.0 + (torch.arange(K) % 8).double()) * (1 - 2 * (torch.arange(K) % 3 == 0).double())).to(BF)
    x[2, :256] = (rand(52, 256).double() * torch.exp2(-90.0 - (torch.arange(256) // 32 * 6).double())).to(BF)
    got = ops.mx4_linear(x.to(cuda), q)
    z, S = x.double() @ w.T, x.double().abs() @ w.abs().T
    blocks = torch.nn.functional.pad(x.double().abs(), (0, -K % 32)).view(M, -1, 32).amax(2).repeat_interleave(32, 1)[:, :K]
    bound = z.abs() * 2.0 ** -8 + S * ((K / 16 + 8) * 2.0 ** -22) + 2.0 ** -31 * (blocks @ w.abs().T) + 2.0 ** -133
    err = (got.double().cpu() - z).abs()
    assert (err <= bound).all(), (err / bound).max().item()


@pytest.mark.parametrize("M, N, four", [(M, 150, four) for M in (3, 40, 300) for four in (False, True)] +
                         [(3, 50000, False), (60, 9000, False), (90, 9000, False), (700, 5000, False)])
def test_not_a_number_stays_in_its_row_and_column(cuda, M, N, four):
    from vila_b200 import ops
    K = 416
    codes, scales = R.quantise(rand(50, N, K))
    scales[17, 3] = 255
    q, w = ops.mx4_pack(codes.to(cuda), scales.to(cuda), K), R.values(codes, scales, K)
    x = rand(51, M, K).to(BF)
    x[1, 200] = math.nan
    x[2, 9] = math.inf
    got = ops.mx4_matmul(ops.mx4_quantize(x.to(cuda)), q) if four else ops.mx4_linear(x.to(cuda), q)
    got = got.float().cpu()
    assert torch.isnan(got[:, 17]).all() and torch.isnan(got[1]).all()
    assert not torch.isfinite(got[2]).any()
    rows = [m for m in range(M) if m not in (1, 2)]
    cols = [n for n in range(N) if n != 17]
    ref = R.values(*R.quantise(x), K) if four else x
    check_product(got[rows][:, cols].to(BF), ref[rows], w[cols], None)


@pytest.mark.parametrize("M, N, K", [(3, 150, 416), (3, 50000, 416), (12, 150, 416), (12, 300, 8200), (40, 150, 416), (60, 9000, 416), (90, 9000, 416),
                                     (700, 5000, 416)])
def test_infinities_and_sums_beyond_the_range(cuda, M, N, K):
    """Whichever kernel takes the rows: products with an infinite entry are infinite, with a weight of 0 NaN, and sums of infinities of both signs
    are NaN.  A sum beyond bf16's largest number is infinite; where the magnitudes add up to less than that, no order of the
    sum leaves the range, and it is held to product_bound.  To that comes what a block's largest entry leaves of the others: the 16 rows that
    an entry is cut into leave 2 units of the last one, 2 * 4^-15 of the first's, which are at most a quarter of the largest: 2^-31
    of it (f16 with a scale per block: 2^-39 of it), times the block's weights."""
    from vila_b200 import ops
    codes, scales = R.quantise(rand(50, N, K))
    codes[::7, 4] &= 0xf0               # column 8: weights of 0
    scales[20, 3] = 255
    q, w = ops.mx4_pack(codes.to(cuda), scales.to(cuda), K), R.values(codes, scales, K)
    x = rand(51, M, K).to(BF)
    x[0, 8] = math.inf
    x[1, 8], x[1, 300] = -math.inf, math.inf
    x[2] = 0
    x[2, 10:14] = torch.tensor([3.3e38, -3.3e38, 3.2e38, 2.0]).to(BF)
    got = ops.mx4_linear(x.to(cuda), q).float().cpu()
    z = torch.stack([(x[m].double() * w).sum(1) for m in range(3)])
    most = (x[2].double().abs() * w.abs()).sum(1)
    assert torch.isnan(got[:, 20]).all()
    assert torch.isinf(z[0]).any() and torch.isnan(z[0]).any() and torch.isinf(z[1]).any()
    assert torch.equal(got[:2].nan_to_num(7.0), z[:2].float().nan_to_num(7.0)) and torch.equal(torch.isnan(got[:2]), torch.isnan(z[:2]))
    inside, beyond = most < 3.3e38, (z[2].abs() == most) & (most > 3.5e38) & torch.isfinite(most)
    assert inside.any() and beyond.any()
    z2, bound = product_bound(x[2:3], w[inside])
    assert ((got[2:3, inside] - z2).abs() <= bound + 2.0 ** -31 * 3.3e38 * w[inside, :32].abs().sum(1)).all()
    assert torch.equal(got[2, beyond].double(), torch.sign(z[2, beyond]) * math.inf)
    cols = [n for n in range(N) if n != 20]
    if M > 3:
        check_product(got[3:][:, cols].to(BF), x[3:], w[cols], None)


@pytest.mark.parametrize("M, N, four", [(M, 384, four) for M in (1, 5, 30, 300) for four in (False, True)] +
                         [(2, 17000, False), (60, 9000, False), (700, 5000, False), (700, 5000, True)])
def test_same_bits_every_time_and_on_another_stream_and_in_a_graph(cuda, M, N, four):
    from vila_b200 import ops
    q, w = weight(60, N, 1000, cuda)
    x = rand(61, M, 1000).to(BF).to(cuda)
    call = (lambda: ops.mx4_matmul(ops.mx4_quantize(x), q)) if four else (lambda: ops.mx4_linear(x, q))
    first = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = call()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, again)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call()
        graphs.append((g, out))
    x2 = rand(62, M, 1000).to(BF).to(cuda)
    x.copy_(x2)
    with torch.cuda.stream(side):       # both replay at once
        side.wait_stream(torch.cuda.current_stream())
        graphs[0][0].replay()
    graphs[1][0].replay()
    torch.cuda.current_stream().wait_stream(side)
    want = call()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1], want) and torch.equal(graphs[1][1], want) and not torch.equal(want, first)
    ops.check_waits()


def test_row_does_not_depend_on_the_rows_around_it_within_a_kernel(cuda):
    from vila_b200 import ops
    q, _ = weight(70, 200, 640, cuda)
    x = rand(71, 6, 640).to(BF).to(cuda)
    got = ops.mx4_linear(x, q)
    x2 = x.clone()
    x2[[0, 1, 2, 4, 5]] = 1e4
    assert torch.equal(ops.mx4_linear(x2, q)[3], got[3])


def product_bound(x, w):
    """|x| . |w| of a bf16 result's rounding (2^-8 of the value) and of the fp32 sums, as in check_product"""
    z, S = x.double() @ w.double().T, x.double().abs() @ w.double().abs().T
    return z, z.abs() * 2.0 ** -8 + S * (x.shape[1] / 16 + 8) * 2.0 ** -22 + 1e-30


@pytest.mark.parametrize("M, N, K", [(270000, 8192, 64), (70000, 512, 32768)])
@pytest.mark.parametrize("four", [False, True])
def test_offsets_past_32_bits(cuda, M, N, K, four):
    """results, and rows, of more than 2^31 elements"""
    from vila_b200 import ops
    x, q = torch.randn(M, K, device=cuda, dtype=BF), ops.mx4_quantize(torch.randn(N, K, device=cuda))
    rows = torch.tensor([0, 1, M // 2, M - 129, M - 1], device=cuda)
    if four:
        a = ops.mx4_quantize(x)
        got, x = ops.mx4_matmul(a, q)[rows], ops.mx4_dequantize(a)[rows]
    else:
        got, x = ops.mx4_linear(x, q)[rows], x[rows]
    z, most = product_bound(x, ops.mx4_dequantize(q, out_dtype=torch.float32))
    assert ((got.double() - z).abs() <= most).all()


@pytest.mark.parametrize("M, N, K", [(8, 500, 32768), (7, 500, 32737), (5, 130, 99999), (3, 129, 60000), (1, 100, 131072), (8, 128, 4096)])
def test_more_columns_than_tokens_fit_in_shared_memory(cuda, M, N, K):
    """few rows, small layers: the tokens of a CTA's part of K come in several portions"""
    from vila_b200 import ops
    x, q = torch.randn(M, K, device=cuda, dtype=BF), ops.mx4_quantize(torch.randn(N, K, device=cuda))
    z, most = product_bound(x, ops.mx4_dequantize(q, out_dtype=torch.float32))
    assert ((ops.mx4_linear(x, q).double() - z).abs() <= most).all()


@pytest.mark.parametrize("M", [1, 8, 9, 16, 17, 40])
@pytest.mark.parametrize("N, K", [(300, 1000), (129, 33000), (3000, 8193)])
@pytest.mark.parametrize("gap", [0, 3])
def test_callers_without_a_workspace(cuda, monkeypatch, M, N, K, gap):
    from vila_b200 import _lib, ops
    x, q = torch.randn(M, K + gap, device=cuda, dtype=BF)[:, :K], ops.mx4_quantize(torch.randn(N, K, device=cuda))
    bias = torch.randn(N, device=cuda, dtype=BF)
    monkeypatch.setattr(_lib.load(), "vila_mx4_linear_scratch", lambda p: 0)
    z, most = product_bound(torch.cat([x, x.new_ones(M, 1)], 1), torch.cat([ops.mx4_dequantize(q, out_dtype=torch.float32), bias.float()[:, None]], 1))
    assert ((ops.mx4_linear(x, q, bias).double() - z).abs() <= most).all()
    ops.check_waits()


@pytest.mark.parametrize("M", [7, 8, 9, 15, 16, 17, 127, 128, 129, 255, 256, 257])
def test_both_sides_of_every_boundary(cuda, M):
    from vila_b200 import ops
    for N in (1, 2, 127, 128, 129, 4096, 4097):
        for K in (1, 31, 32, 33, 255, 256, 257, 4096):
            x, q = torch.randn(M, K, device=cuda, dtype=BF), ops.mx4_quantize(torch.randn(N, K, device=cuda))
            z, most = product_bound(x, ops.mx4_dequantize(q, out_dtype=torch.float32))
            assert ((ops.mx4_linear(x, q).double() - z).abs() <= most).all(), (N, K)


def test_four_streams_at_once(cuda):
    from vila_b200 import ops
    q = ops.mx4_quantize(torch.randn(9000, 1000, device=cuda))
    xs = [torch.randn(m, 1000, device=cuda, dtype=BF) for m in (2, 12, 60, 700)]
    want = [ops.mx4_linear(x, q) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    for _ in range(20):
        got = []
        for x, stream in zip(xs, streams):
            with torch.cuda.stream(stream):
                got.append(ops.mx4_linear(x, q))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    ops.check_waits()


FIRST_CALLS = """
import threading, torch
from vila_b200 import ops
torch.manual_seed(0)
cases = [(1, 2000, 2000, False), (8, 9000, 4000, False), (16, 3584, 4096, False), (60, 12000, 520, False), (90, 12000, 520, False), (1200, 5000, 520, False),
         (16, 300, 8192, True), (100, 300, 5000, True), (300, 514, 800, True), (1500, 1300, 800, True)]
data = [(torch.randn(M, K, device="cuda").bfloat16(), ops.mx4_quantize(torch.randn(N, K, device="cuda")), four) for M, N, K, four in cases]
torch.cuda.synchronize()
def call(x, w, four):
    return ops.mx4_matmul(ops.mx4_quantize(x), w) if four else ops.mx4_linear(x, w)
got, errors, threads = [[None] * len(data) for _ in range(8)], [], []
start = threading.Barrier(8)
def work(t):
    try:
        with torch.cuda.stream(torch.cuda.Stream()):
            for i in range(len(data)):
                start.wait()
                got[t][i] = call(*data[i])
            torch.cuda.current_stream().synchronize()
    except Exception as e:
        errors.append(repr(e))
        start.abort()
for t in range(8):
    threads.append(threading.Thread(target=work, args=(t,)))
    threads[-1].start()
for t in threads:
    t.join()
assert not errors, errors
torch.cuda.synchronize()
for i, d in enumerate(data):
    want = call(*d)
    assert all(torch.equal(g[i], want) for g in got), i
ops.check_waits()
print("agree")
"""


def test_first_calls_from_several_host_threads(cuda):
    """every kernel's first launch of a process comes from eight threads at once: none is refused, and all cut K alike"""
    import subprocess
    import sys
    from pathlib import Path
    root = Path(__file__).resolve().parent.parent
    r = subprocess.run([sys.executable, "-c", FIRST_CALLS], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "agree" in r.stdout, r.stdout + r.stderr


def test_no_rows(cuda):
    from vila_b200 import ops
    q, _ = weight(80, 64, 64, cuda)
    assert ops.mx4_linear(torch.empty(0, 64, dtype=BF, device=cuda), q).shape == (0, 64)
    assert ops.mx4_matmul(ops.mx4_quantize(torch.empty(0, 64, device=cuda)), q, swiglu=True).shape == (0, 32)


def test_refusals(cuda):
    from vila_b200 import ops
    q, _ = weight(90, 65, 64, cuda)
    x = torch.zeros(4, 64, dtype=BF, device=cuda)
    for match, call in [
        ("do not fit a weight", lambda: ops.mx4_linear(x[:, :32], q)),
        ("must be torch.bfloat16", lambda: ops.mx4_linear(x.float(), q)),
        ("must be an Mx4", lambda: ops.mx4_linear(x, x)),
        ("consecutive columns", lambda: ops.mx4_linear(torch.zeros(64, 4, dtype=BF, device=cuda).T, q)),
        ("even number of weight rows", lambda: ops.mx4_linear(x, q, swiglu=True)),
        ("one gated unit", lambda: ops.mx4_linear(x, q, swiglu=True, geglu=True)),
        ("unknown activation", lambda: ops.mx4_linear(x, q, act=ops.ACT_SOFTCAP)),
        ("takes act_params", lambda: ops.mx4_linear(x, q, act=ops.ACT_XIELU)),
        ("bias must be", lambda: ops.mx4_linear(x, q, torch.zeros(65, device=cuda))),
        ("bias must be", lambda: ops.mx4_linear(x, q, torch.zeros(64, dtype=BF, device=cuda))),
        ("out must be", lambda: ops.mx4_linear(x, q, out=torch.zeros(4, 64, dtype=BF, device=cuda))),
        ("consecutive columns", lambda: ops.mx4_quantize(torch.zeros(64, 4, device=cuda).T)),
        ("bfloat16 or float32", lambda: ops.mx4_quantize(torch.zeros(4, 64, device=cuda, dtype=torch.float16))),
        ("bfloat16 or float32", lambda: ops.mx4_dequantize(q, out_dtype=torch.float16)),
        ("scales must be", lambda: ops.mx4_pack(q.codes, torch.zeros(65, 3, dtype=torch.uint8, device=cuda), 64)),
    ]:
        with pytest.raises(RuntimeError, match=match):
            call()
    gated, _ = weight(91, 64, 64, cuda)
    with pytest.raises(RuntimeError, match="takes no other activation"):
        ops.mx4_linear(x, gated, swiglu=True, act=ops.ACT_SILU)


def test_pointers_that_are_refused_on_the_host(cuda):
    """null pointers, and pointers off their elements' boundaries, reach no kernel"""
    import ctypes as C
    from vila_b200 import _lib, ops
    lib = _lib.load()
    q, _ = weight(92, 4, 64, cuda)
    x = torch.zeros(4, 64, device=cuda)
    codes, scales, at = q.codes.data_ptr(), q.scales.data_ptr(), x.data_ptr()
    BF16, F32 = ops._dt(x.to(BF), "x"), ops._dt(x, "x")
    for refused in (lib.vila_mx4_quantize(None, F32, 64, codes, scales, 4, 64, None), lib.vila_mx4_quantize(at + 2, F32, 64, codes, scales, 3, 64, None),
                    lib.vila_mx4_quantize(at + 1, BF16, 64, codes, scales, 3, 64, None), lib.vila_mx4_quantize(at, F32, 64, None, scales, 4, 64, None),
                    lib.vila_mx4_dequantize(codes, scales, None, F32, 64, 4, 64, None), lib.vila_mx4_dequantize(codes, scales, at + 2, F32, 64, 3, 64, None),
                    lib.vila_mx4_dequantize(codes, scales, at, F32, 63, 4, 64, None), lib.vila_mx4_dequantize(codes, None, at, F32, 64, 4, 64, None),
                    lib.vila_mx4_scales(None, scales, 4, 64, 0, None), lib.vila_mx4_scales(at, None, 4, 64, 0, None)):
        assert refused == 1
    good = dict(x=at, ldx=64, w_codes=codes, w_scales=scales, out=at, ldo=4, M=4, N=4, K=64)
    for bad in (dict(x=None), dict(x=at + 1), dict(out=None), dict(out=at + 1), dict(bias=at + 1), dict(w_codes=None), dict(w_scales=None),
                dict(x=None, a_codes=codes), dict(w_codes=codes + 8), dict(ldo=3)):
        assert lib.vila_mx4_linear(C.byref(_lib.Mx4LinearParams(**{**good, **bad})), None) == 1, bad
    assert lib.vila_mx4_linear(None, None) == 1 and lib.vila_mx4_linear_tries(None, 5, None) == 1
    assert lib.vila_mx4_quantize(None, F32, 64, None, None, 0, 64, None) == 0      # no rows, nothing to point at
    torch.cuda.synchronize()
    assert not x.any()


# ---- waits that run out ----------------------------------------------------------------------------------
# rows, weight rows, columns, 4-bit rows: one for every tcgen05 kernel and tile
KERNELS = [(16, 300, 800, True), (40, 300, 800, True), (100, 300, 5000, True), (300, 514, 800, True), (1500, 1300, 800, True),
           (12, 300, 4800, False), (40, 2600, 520, False), (60, 12000, 520, False), (90, 12000, 520, False), (120, 12000, 520, False),
           (1200, 5000, 520, False)]


@pytest.mark.parametrize("tries", [0, 1, 30, -2, -3, -4, -5])
@pytest.mark.parametrize("M, N, K, four", KERNELS)
def test_waits_that_run_out(cuda, monkeypatch, M, N, K, four, tries):
    """The launch ends, the next status says so once, and the call after that is right."""
    from vila_b200 import _lib, ops
    w = ops.mx4_quantize(torch.randn(N, K, device=cuda, generator=torch.Generator(cuda).manual_seed(1)))
    x = torch.randn(M, K, device=cuda, generator=torch.Generator(cuda).manual_seed(2)).to(BF)
    call = (lambda: ops.mx4_matmul(ops.mx4_quantize(x), w)) if four else (lambda: ops.mx4_linear(x, w))
    want = call()
    torch.cuda.synchronize()
    ops.check_waits()
    lib = _lib.load()
    with monkeypatch.context() as m:
        m.setattr(lib, "vila_mx4_linear", lambda p, stream: lib.vila_mx4_linear_tries(p, tries, stream))
        out = call()
        torch.cuda.synchronize()
    unpacks = not four and M > 16 and -(-N // 128) * -(-M // 8) > 2 * torch.cuda.get_device_properties(0).multi_processor_count
    if tries == 0 or (tries < 0 and (tries != -4 or unpacks)) or not torch.equal(out, want):
        with pytest.raises(RuntimeError, match="ran out of tries"):
            ops.check_waits()
    else:
        try:      # a warp may have given up behind the last wait that its output needs
            ops.check_waits()
        except RuntimeError:
            pass
    ops.check_waits()
    assert torch.equal(call(), want)


@pytest.mark.parametrize("role", [0, 1, 2, 3])
@pytest.mark.parametrize("rank", [0, 1])
@pytest.mark.parametrize("M, N, K, four", [(1500, 1300, 800, True), (1500, 1300, 5000, True), (1200, 5000, 520, False), (1200, 5000, 5000, False)])
def test_one_cta_of_a_pair_gives_up(cuda, monkeypatch, M, N, K, four, rank, role):
    """One CTA of every pair quits while the other has copies in flight that report to it, or expects copies that the first has not
    asked for: the launch ends, says so, and the calls after it are right."""
    from vila_b200 import _lib, ops
    w = ops.mx4_quantize(torch.randn(N, K, device=cuda, generator=torch.Generator(cuda).manual_seed(1)))
    x = torch.randn(M, K, device=cuda, generator=torch.Generator(cuda).manual_seed(2)).to(BF)
    call = (lambda: ops.mx4_matmul(ops.mx4_quantize(x), w)) if four else (lambda: ops.mx4_linear(x, w))
    want = call()
    torch.cuda.synchronize()
    ops.check_waits()
    lib = _lib.load()
    for _ in range(3):
        with monkeypatch.context() as m:
            m.setattr(lib, "vila_mx4_linear", lambda p, stream: lib.vila_mx4_linear_tries(p, -2 - (role + 4 * (rank + 1)), stream))
            out = call()
            torch.cuda.synchronize()
        if (four and role == 2) or (rank == 1 and role == 1):      # no such warp: unpacking, the second CTA's products
            assert torch.equal(out, want)
        else:
            with pytest.raises(RuntimeError, match="ran out of tries"):
                ops.check_waits()
        ops.check_waits()
        assert torch.equal(call(), want)


def test_nothing_is_launched_behind_a_launch_that_gave_up(cuda, monkeypatch):
    from vila_b200 import _lib, ops
    w = ops.mx4_quantize(torch.randn(300, 800, device=cuda))
    a = ops.mx4_quantize(torch.randn(40, 800, device=cuda))
    lib = _lib.load()
    with monkeypatch.context() as m:
        m.setattr(lib, "vila_mx4_linear", lambda p, stream: lib.vila_mx4_linear_tries(p, 0, stream))
        ops.mx4_matmul(a, w)
    torch.cuda.synchronize()
    out = torch.full((40, 300), 7.0, dtype=BF, device=cuda)
    with pytest.raises(RuntimeError, match="ran out of tries"):
        ops.mx4_matmul(a, w, out=out)
    torch.cuda.synchronize()
    assert (out == 7).all()
    ops.mx4_matmul(a, w, out=out)


# ---- together, as they are used -----------------------------------------------------------------------------
@pytest.mark.parametrize("M", [1, 12, 40, 300])
def test_feed_forward_block(cuda, M):
    """gate / up with a gated unit, then down, on weights in 4 bits: rows as they come, and quantised before each product"""
    from vila_b200 import ops
    gu, gu64 = weight(100, 512, 384, cuda)
    down, down64 = weight(102, 384, 256, cuda)
    x = rand(104, M, 384).to(BF).to(cuda)
    h = ops.linear_any(x, gu, swiglu=True)
    check_product(h, x, gu64, None, "swiglu")
    check_product(ops.linear_any(h, down), h, down64, None)
    q = ops.mx4_quantize(x)
    h = ops.mx4_matmul(q, gu, swiglu=True)
    check_product(h, ops.mx4_dequantize(q, out_dtype=torch.float32), gu64, None, "swiglu")
    hq = ops.mx4_quantize(h)
    check_product(ops.mx4_matmul(hq, down), ops.mx4_dequantize(hq, out_dtype=torch.float32), down64, None)
    with pytest.raises(RuntimeError, match="gives bfloat16"):
        ops.linear_any(x, gu, out_dtype=torch.float32)
    with pytest.raises(RuntimeError, match="must be torch.bfloat16"):
        ops.linear_any(x.float(), gu)


@pytest.mark.parametrize("arch", ["nusovik", "ludazen", "bivizen", "nibelix", "lufatar"])
def test_language_models_on_4_bit_weights(cuda, arch):
    """A model whose layers' weights are in 4 bits against the same model with the bf16 weights that these stand for (each is a bf16
    number): prompts, portions and decoded tokens, eager and captured.  The projections' sums differ by fp32 rounding alone, so that
    a bf16 rounding may fall the other way: the whole models agree to the bound that they are held to against their oracles."""
    import importlib
    from vila_b200 import ops
    from vila_b200.model.registry import MX4_WEIGHTS, quantize_weights
    from vila_b200.serving import TokenEngine
    T = importlib.import_module(f"tests.test_{arch}_gpu")
    name = "aligned" if "aligned" in T.CONFIGS else next(iter(T.CONFIGS))
    cfg, small = T.build(name, BF, seed=3)
    _, plain = T.build(name, BF, seed=3)
    before = {k: v.clone() for k, v in small.state_dict().items()}
    assert quantize_weights(small) is small
    held = 0
    for a, b in zip(small.layers, plain.layers):
        for n in MX4_WEIGHTS[type(small).__name__.replace("ForCausalLM", "")]:
            q = getattr(a, n, None)
            if isinstance(q, ops.Mx4):
                held += 1
                setattr(b, n, ops.mx4_dequantize(q))
    assert held >= len(small.layers)
    assert all(torch.equal(v, before[k]) for k, v in small.state_dict().items())
    ea, eb = TokenEngine(small, 256, 2), TokenEngine(plain, 256, 2)
    toks = T.tokens_for(cfg, 60, 5)
    for entries in ([("a", toks[:40], [0, 39]), ("b", toks[:7], [6])], [("a", toks[40:41], [0]), ("b", toks[7:30], [22])],
                    *[[("a", [toks[41 + i]], [0]), ("b", [toks[30 + i]], [0])] for i in range(4)]):
        got, want = ea.step(entries), eb.step(entries)
        assert ((got - want).abs().max() / want.abs().max()).item() < 5e-2
    assert len(small.generate(toks[:9], max_new_tokens=5)[0]) == 5


@pytest.mark.parametrize("arch", ["nusovik", "ludazen", "bivizen", "nibelix", "lufatar"])
def test_weights_replaced_under_an_engine_that_has_captured_its_steps(cuda, arch):
    """quantize_weights, then load_weights, between decoded tokens: an engine with graphs goes on as one without."""
    import importlib
    from vila_b200.model.registry import quantize_weights
    from vila_b200.serving import TokenEngine
    T = importlib.import_module(f"tests.test_{arch}_gpu")
    name = "aligned" if "aligned" in T.CONFIGS else next(iter(T.CONFIGS))
    cfg, model = T.build(name, BF, seed=3)
    loaded = dict(model.state_dict())
    engines = [TokenEngine(model, 256, 2), TokenEngine(model, 256, 2, graphs=False)]
    toks = T.tokens_for(cfg, 60, 5)
    both = [[] for _ in engines]

    def decode(first, n):
        for e, got in zip(engines, both):
            for t in toks[first:first + n]:
                got.append(e.step([("a", [t], [0])]))

    for e in engines:
        e.step([("a", toks[:20], [19])])
    decode(20, 4)
    assert engines[0]._decode_graphs
    quantize_weights(model)
    decode(24, 4)
    assert engines[0]._decode_graphs
    model.load_weights(loaded)
    decode(28, 4)
    assert all(torch.equal(a, b) for a, b in zip(*both))


@pytest.mark.parametrize("arch, layer_type, name", [("bivizen", "delta", "in_w"), ("bivizen", "gla", "in_w"), ("nusovik", "parallel", "ssd_in")])
def test_rows_of_decays_and_step_sizes_stay_exact(cuda, arch, layer_type, name):
    """The rows that a recurrence's decay and step size come from keep the weights that were loaded, and their columns of the projection are
    those of the bf16 model to the bound of one linear layer; the rows before them are in 4 bits."""
    import importlib
    from vila_b200 import ops
    from vila_b200.model.registry import quantize_weights
    T = importlib.import_module(f"tests.test_{arch}_gpu")
    cfg, small = T.build("aligned" if "aligned" in T.CONFIGS else next(iter(T.CONFIGS)), BF, seed=3)
    loaded = small.state_dict()
    before = [getattr(L, name, None) for L in small.layers]
    quantize_weights(small)
    seen = 0
    for i, (L, w) in enumerate(zip(small.layers, before)):
        if L.cfg.type != layer_type:
            continue
        seen += 1
        if arch == "bivizen":
            parts = ("a", "b") if layer_type == "delta" else ("a1",)
            exact = [(L.in_off[n], loaded[f"l{i}.mix.{n}"]) for n in parts]
        else:
            r = L.cfg.right
            exact = [((r.inner + r.conv_channels, r.heads), loaded[f"l{i}.mix.right.in"][r.inner + r.conv_channels:])]
        held = ops.mx4_dequantize(getattr(L, name))
        first = exact[0][0][0]
        x = rand(i, 5, w.shape[1]).to(BF)
        got = ops.linear_any(x.to(cuda), getattr(L, name))
        for (at, n), want in exact:
            want = want.to(cuda, BF)
            assert torch.equal(held[at:at + n], want) and torch.equal(w[at:at + n], want)
            check_product(got[:, at:at + n], x, want, None)
        assert torch.equal(held[first:], w[first:])
        rows = first // 8 * 8
        assert torch.equal(held[:rows], ops.mx4_dequantize(ops.mx4_quantize(w[:rows]))) and not torch.equal(held[:rows], w[:rows])
        check_product(got, x, held, None)
    assert seen


@pytest.mark.parametrize("M", [0, 1, 12, 60, 700])
@pytest.mark.parametrize("N, keep, K", [(200, 8, 288), (200, 7, 288), (96, 64, 100), (2, 1, 32), (640, 320, 512)])
def test_rows_that_stay_as_they_are(cuda, M, N, keep, K):
    from vila_b200 import ops
    w, x, bias = (rand(1, N, K) / math.sqrt(K)).to(BF), rand(2, M, K).to(BF), rand(3, N).to(BF)
    q = ops.mx4_quantize(w.to(cuda), keep=keep)
    assert q.shape == (N, K) and q.device == x.to(cuda).device and q.nbytes == q.part.nbytes + keep * K * 2
    both = ops.mx4_dequantize(q).cpu()
    assert torch.equal(both[N - keep:], w[N - keep:]) and torch.equal(both[:N - keep], ops.mx4_dequantize(ops.mx4_quantize(w[:N - keep].to(cuda))).cpu())
    assert torch.equal(ops.mx4_dequantize(q, out_dtype=torch.float32).cpu(), both.float())
    out = torch.full((M, N + 5), 7.0, dtype=BF, device=cuda)
    check = check_product if M else lambda got, *rest: None
    check(ops.mx4_linear(x.to(cuda), q, bias.to(cuda), out=out[:, 2:2 + N]), x, both, bias)
    assert (out[:, :2] == 7).all() and (out[:, 2 + N:] == 7).all()
    check(ops.linear_any(x.to(cuda), q, act=ops.ACT_SILU), x, both, None, "silu")
    if N % 2 == 0 and keep % 2 == 0:
        check(ops.linear_any(x.to(cuda), q, bias=bias.to(cuda), swiglu=True), x, both, bias, "swiglu")
    elif M:
        with pytest.raises(RuntimeError, match="even number of weight rows"):
            ops.linear_any(x.to(cuda), q, swiglu=True)


@pytest.mark.parametrize("M", [1, 12, 300])
def test_rows_that_stay_as_they_are_under_views_and_broadcast_rows(cuda, M):
    from vila_b200 import ops
    N, K, keep = 200, 288, 24
    w = (rand(1, N, K) / math.sqrt(K)).to(BF)
    q = ops.mx4_quantize(w.to(cuda), keep=keep)
    both = ops.mx4_dequantize(q)
    for gap, off in ((8, 0), (3, 0), (8, 1), (0, 2), (8, 8)):
        wide = rand(2, M, K + gap + off).to(BF).to(cuda)
        check_product(ops.mx4_linear(wide[:, off:off + K], q), wide[:, off:off + K], both, None)
    one = rand(3, 1, K).to(BF).to(cuda).expand(M, K)
    check_product(ops.linear_any(one, q), one, both, None)
    if M == 1:
        column, out = torch.empty(K, 1, dtype=BF, device=cuda), torch.empty(N, 1, dtype=BF, device=cuda)
        column.copy_(one.T)
        check_product(ops.mx4_linear(column.T, q, out=out.T), one, both, None)
        assert out.any()


def test_rows_kept_in_bf16_are_refused_where_codes_are_read(cuda):
    from vila_b200 import ops
    w = rand(1, 64, 64).to(BF).to(cuda)
    q, a = ops.mx4_quantize(w, keep=8), ops.mx4_quantize(w)
    for call in (lambda: ops.mx4_matmul(a, q), lambda: ops.mx4_matmul(q, a), lambda: ops.mx4_unpack(q), lambda: q.codes, lambda: q.scales):
        with pytest.raises(RuntimeError, match="kept in bf16"):
            call()
    for bad in (64, 65, -1):
        with pytest.raises(RuntimeError, match="not all of them"):
            ops.mx4_quantize(w, keep=bad)
    with pytest.raises(RuntimeError, match="not all of them"):
        ops.mx4_quantize(w.float(), keep=8)


def test_load_and_command_line(cuda, tmp_path, capsys):
    from llava.cli import infer
    from tests import test_nusovik_gpu as T
    from vila_b200 import ops
    from vila_b200.model import load_language_model
    cfg, model = T.build("aligned", BF, seed=8)
    model.save_pretrained(tmp_path / "m")
    small = load_language_model(tmp_path / "m", weights="mx4")
    assert isinstance(small.layers[0].sel_in, ops.Mx4)
    prompt = T.tokens_for(cfg, 9, 4)
    text = infer.main(["--model-path", str(tmp_path / "m"), "--token-ids", ",".join(map(str, prompt)), "--max-new-tokens", "5", "--weights", "mx4"])
    assert [int(t) for t in text.split(",")] == small.generate(prompt, max_new_tokens=5)[0]
    assert text in capsys.readouterr().out
