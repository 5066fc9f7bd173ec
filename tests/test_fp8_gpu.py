"""GPU: 8-bit rows with a scale per block of 128 against their restatement in float64."""
import ctypes as C
import gc
import math

import pytest
import torch

from tests import fp8_reference as R
from tests.test_mx4_gpu import act64, act_args, check_product

pytestmark = pytest.mark.gpu
BF, E4M3 = torch.bfloat16, torch.float8_e4m3fn


@pytest.fixture(autouse=True)
def nothing_left_behind():
    """Models and their captured steps refer to one another: they go here, and not while a later test captures."""
    yield
    gc.collect()


def rand(seed, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def same(q, x, block_rows=1):
    """q is the 8-bit form of x, bit by bit"""
    codes, scales = R.quantise(x, block_rows)
    assert q.shape == tuple(x.shape) and q.codes.dtype == E4M3 and q.scales.dtype == torch.float32 and q.scales.shape == scales.shape
    assert torch.equal(q.codes.cpu().double(), codes)
    assert torch.equal(q.scales.cpu().nan_to_num(-1.0), scales.nan_to_num(-1.0))


# ---- quantisation: bit by bit -------------------------------------------------------------------------
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("rows, cols", [(1, 1), (1, 15), (1, 16), (3, 17), (2, 127), (129, 128), (5, 129), (130, 1000), (257, 256), (7, 3584), (300, 401)])
def test_quantise_is_the_definition(cuda, rows, cols, dtype, block_rows):
    from vila_b200 import ops
    x = (rand(1, rows, cols) * torch.exp(2 * rand(2, 1, cols))).to(dtype)
    q = ops.fp8_quantize(x.to(cuda), block_rows=block_rows)
    same(q, x, block_rows)
    want = R.values(*R.quantise(x, block_rows), block_rows)
    assert torch.equal(ops.fp8_dequantize(q, out_dtype=torch.float32).cpu(), want.float())      # one rounding of the product
    assert torch.equal(ops.fp8_dequantize(q).cpu(), want.float().to(BF))


def test_every_number_comes_back(cuda):
    from vila_b200 import ops
    codes = torch.arange(256, dtype=torch.uint8).view(E4M3).view(2, 128)
    q = ops.fp8_pack(codes.to(cuda), torch.tensor([[1.0], [2.0]], device=cuda), block_rows=1)
    got = ops.fp8_dequantize(q, out_dtype=torch.float32).cpu()
    want = codes.float() * torch.tensor([[1.0], [2.0]])
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0))


@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantise_edges(cuda, block_rows):
    from vila_b200 import ops
    x = torch.zeros(12 * block_rows, 256)
    at = x[::block_rows]
    ties = torch.tensor([448.0, 17.0, 19.0, -17.0, -19.0, 2.0 ** -10, 3 * 2.0 ** -10, -0.0, 0.0, 447.9, 432.0, 440.0, 1.0625, -1.1875])
    at[0, :14] = ties
    at[1, :14] = ties * 2.0 ** 100
    at[2, :14] = ties * 2.0 ** -120
    at[3, :4] = torch.tensor([2.0 ** -149, 2.0 ** -140, 0.0, -(2.0 ** -130)])        # fp32 subnormals
    at[4, 128:132] = torch.tensor([3.4028234e38, -3.4028234e38, 1e38, 1.0])
    at[5, 3] = math.inf
    at[6, 140] = math.nan
    at[7, 3], at[7, 4] = math.nan, -math.inf
    at[8] = 6.0
    at[9, 0] = 2.0 ** -126 * 448
    at[10, 0] = 2.0 ** -125 * 448
    at[11] = -1e-45
    q = ops.fp8_quantize(x.to(cuda), block_rows=block_rows)
    same(q, x, block_rows)
    back = ops.fp8_dequantize(q, out_dtype=torch.float32).cpu()[::block_rows]
    assert back[5, :128].isnan().all() and not back[5, 128:].isnan().any() and back[6, 128:].isnan().all() and back[7, :128].isnan().all()
    assert back.isnan().sum() == 3 * 128


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("gap, off", [(16, 0), (8, 0), (3, 0), (8, 1), (0, 3), (8, 8)])
def test_quantise_views(cuda, gap, off, dtype, block_rows):
    from vila_b200 import ops
    wide = rand(3, 140, 300 + gap + off).to(dtype)
    same(ops.fp8_quantize(wide.to(cuda)[:, off:off + 300], block_rows=block_rows), wide[:, off:off + 300], block_rows)


def test_quantise_broadcast_rows_one_column_and_no_rows(cuda):
    from vila_b200 import ops
    x = rand(4, 1, 96)
    for block_rows in (1, 128):
        same(ops.fp8_quantize(x.to(cuda).expand(5, 96), block_rows=block_rows), x.expand(5, 96), block_rows)
        same(ops.fp8_quantize(rand(5, 7, 9).to(cuda)[:, 4:5], block_rows=block_rows), rand(5, 7, 9)[:, 4:5], block_rows)
        none = ops.fp8_quantize(torch.empty(0, 96, device=cuda), block_rows=block_rows)
        assert none.shape == (0, 96) and none.codes.shape == (0, 96) and none.scales.shape == (0, 1) and ops.fp8_dequantize(none).shape == (0, 96)


def test_pack_keeps_what_lies_well_and_copies_the_rest(cuda):
    from vila_b200 import ops
    codes, scales = (rand(6, 200, 288) * 50).to(E4M3).to(cuda), rand(7, 2, 3).abs().to(cuda)
    want = R.values(codes.cpu().double(), scales.cpu(), 128).float()
    q = ops.fp8_pack(codes, scales)
    assert q.codes.data_ptr() == codes.data_ptr() and q.scales.data_ptr() == scales.data_ptr()
    odd = codes.new_empty(200, 291)
    odd[:, 2:290] = codes
    inner = codes.new_empty(200, 320)
    inner[:, 16:304] = codes
    for c, s, kept in ((odd[:, 2:290], scales, False), (codes.T.contiguous().T, scales, False), (codes, scales.T.contiguous().T, True),
                       (inner[:, 16:304], scales, True)):
        q = ops.fp8_pack(c, s)
        assert (q.codes.data_ptr() == c.data_ptr()) == kept
        assert torch.equal(ops.fp8_dequantize(q, out_dtype=torch.float32).cpu(), want)
    rows = rand(8, 200, 3).abs().to(cuda)       # a scale per row
    q = ops.fp8_pack(codes, rows, block_rows=1)
    assert q.codes.data_ptr() == codes.data_ptr()
    assert torch.equal(q.scales, rows) and torch.equal(ops.fp8_dequantize(q, out_dtype=torch.float32).cpu(), R.values(codes.cpu().double(), rows.cpu(), 1).float())
    for n, k in ((1, 17), (1, 300), (3, 1), (0, 40), (5, 128)):
        few, per = (rand(9, n, k) * 50).to(E4M3).to(cuda), rand(10, n, -(-k // 128)).abs().to(cuda)
        p = ops.fp8_pack(few, per, block_rows=1)
        assert p.shape == (n, k) and torch.equal(p.scales, per) and torch.equal(p.codes.float(), few.float())
        assert torch.equal(ops.fp8_dequantize(p, out_dtype=torch.float32).cpu(), R.values(few.cpu().double(), per.cpu(), 1).float())
    again = ops.fp8_pack(q.codes, q.scales, block_rows=1)
    assert again.scales.data_ptr() == q.scales.data_ptr() and again.codes.data_ptr() == q.codes.data_ptr()


# ---- the norm ----------------------------------------------------------------------------------------------
def check_norm(q, x, w, eps):
    """q against quantise(x / sqrt(mean(x^2) + eps) * w) in float64.  The sum of squares: a thread adds at most 64 squares one after another
    and 10 sums join, each rounded (2^-24): 75 roundings, half of that behind the root; mean, eps, root, reciprocal, two products and
    the format's quotients and product: 9 more.  d = 48 * 2^-24 relative.  Then the number: half a step, 2^-4 of it, or of those below
    2^-6 2^-10, in units of the scale."""
    x = x.double().cpu()
    y = x / torch.sqrt((x * x).mean(1, keepdim=True) + eps)
    if w is not None:
        y = y * w.double().cpu()
    d = 48 * 2.0 ** -24
    top = torch.from_numpy(abs(R.blocks(y.numpy(), 1)).max((1, 3)))
    scales = q.scales.cpu().double()
    want = (top / 448).clamp(min=2.0 ** -126)
    assert scales.shape == want.shape and ((scales - want).abs() <= want * (d + 2.0 ** -23)).all()
    s = R.per_element(scales, 1, *y.shape)
    v = q.codes.cpu().double() * s
    assert ((v - y).abs() <= torch.maximum(v.abs() * 2.0 ** -4, s * 2.0 ** -10) * (1 + 2 * d) + y.abs() * d).all()


@pytest.mark.parametrize("dtype, r_dtype, w_dtype", [(BF, BF, BF), (torch.float32, BF, torch.float32), (BF, torch.float32, None), (torch.float32, torch.float32, BF)])
@pytest.mark.parametrize("rows, cols", [(1, 1), (1, 3584), (3, 17), (70, 128), (5, 1153), (9, 4301), (2, 8192), (2, 8209), (2, 16384), (3, 18944), (2, 32768)])
def test_norm(cuda, rows, cols, dtype, r_dtype, w_dtype):
    from vila_b200 import ops
    x, r = (3 * rand(10, rows, cols) * torch.exp(rand(11, 1, cols))).to(dtype), rand(12, rows, cols).to(r_dtype)
    w = None if w_dtype is None else (1 + 0.2 * rand(13, cols)).to(w_dtype)
    xc, rc, wc = x.to(cuda), r.to(cuda), None if w is None else w.to(cuda)
    q, s = ops.fp8_rmsnorm(xc, wc, 1e-6)
    assert s is xc and torch.equal(xc.cpu(), x)
    check_norm(q, x, w, 1e-6)
    total = (x.float() + r.float()).to(dtype)
    q, s = ops.fp8_rmsnorm(xc, wc, 1e-6, residual=rc)
    assert torch.equal(s.cpu(), total) and torch.equal(xc.cpu(), x) and torch.equal(rc.cpu(), r)
    check_norm(q, total, w, 1e-6)
    same_codes, same_scales = q.codes.clone(), q.scales.clone()
    q, s = ops.fp8_rmsnorm(xc, wc, 1e-6, residual=rc, out=xc)
    assert s is xc and torch.equal(xc.cpu(), total) and torch.equal(q.codes.float(), same_codes.float()) and torch.equal(q.scales, same_scales)


@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("gap, off", [(16, 0), (8, 8), (3, 0), (0, 1)])
def test_norm_of_views(cuda, gap, off, dtype):
    from vila_b200 import ops
    cols = 520
    wide, more, w = rand(14, 33, cols + gap + off).to(dtype), rand(15, 33, cols + gap + off).to(BF), rand(16, cols + 1).to(BF)
    out = torch.full((33, cols + gap + off + 2), 7.0, dtype=dtype, device=cuda)
    view = slice(off, off + cols)
    q, s = ops.fp8_rmsnorm(wide.to(cuda)[:, view], w.to(cuda)[1:], 1e-5, residual=more.to(cuda)[:, view], out=out[:, 1:1 + cols])
    total = (wide[:, view].float() + more[:, view].float()).to(dtype)
    assert torch.equal(s.cpu(), total) and s.data_ptr() == out[:, 1:].data_ptr() and (out[:, :1] == 7).all() and (out[:, 1 + cols:] == 7).all()
    check_norm(q, total, w[1:], 1e-5)
    one = rand(17, 1, cols).to(dtype)
    check_norm(ops.fp8_rmsnorm(one.to(cuda).expand(6, cols), None, 1e-5)[0], one.expand(6, cols), None, 1e-5)


def test_norm_of_zeros_infinities_and_nan(cuda):
    from vila_b200 import ops
    x = rand(18, 5, 300)
    x[0] = 0
    x[1, 200] = math.nan
    x[2, 5] = math.inf
    x[3] = 0
    x[3, 299] = 1e-30
    q, _ = ops.fp8_rmsnorm(x.to(cuda), None, 0.0)
    back = ops.fp8_dequantize(q, out_dtype=torch.float32).cpu()
    assert back[0].isnan().all() and back[1].isnan().all()              # 0 / 0 with eps = 0, as the formula has it
    assert back[2, :128].isnan().all() and (back[2, 128:] == 0).all()   # infinity / infinity, and what is divided by infinity
    check_norm(ops.fp8_rmsnorm(x[4:].to(cuda), None, 0.0)[0], x[4:], None, 0.0)
    zero = ops.fp8_rmsnorm(torch.zeros(3, 200, device=cuda), None, 1e-6)[0]
    assert (ops.fp8_dequantize(zero) == 0).all() and (zero.scales == 2.0 ** -126).all()
    assert ops.fp8_rmsnorm(torch.empty(0, 200, device=cuda), None, 1e-6)[0].shape == (0, 200)


# ---- products --------------------------------------------------------------------------------------------
def weight(seed, n, k, cuda, spread=0.0):
    from vila_b200 import ops
    w = rand(seed, n, k) / math.sqrt(k) * torch.exp(spread * rand(seed + 1, n, 1))
    codes, scales = R.quantise(w, 128)
    return ops.fp8_pack(codes.to(E4M3).to(cuda), scales.to(cuda)), R.values(codes, scales, 128)


def rows8(x, cuda):
    """8-bit rows of x and what they stand for"""
    from vila_b200 import ops
    codes, scales = R.quantise(x, 1)
    return ops.fp8_pack(codes.to(E4M3).to(cuda), scales.to(cuda), block_rows=1), R.values(codes, scales, 1)


def check_rows8(q, x, w, bias, act="none"):
    """q (Fp8) against quantise(act(x w^T + bias)) in float64: check_product's bound for the sums and the activation (without the
    rounding to bf16), then the format's own half step."""
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
    off = 2 * off + want.abs() * 2.0 ** -20
    if act in ("gelu_tanh", "gelu_erf"):
        off = off + z.abs() * 2.0 ** -22
    elif act in ("geglu", "glu_clamp"):
        off = off + z[:, 0::2].abs() * (z[:, 1::2].abs() + 1) * 2.0 ** -22
    top, most = (torch.from_numpy(abs(R.blocks(t.numpy(), 1)).max((1, 3))) for t in (want, off))
    scales = q.scales.cpu().double()
    assert q.shape == tuple(want.shape) and ((scales - (top / 448).clamp(min=2.0 ** -126)).abs() <= most / 448 + top / 448 * 2.0 ** -23).all()
    s = R.per_element(scales, 1, *want.shape)
    v = q.codes.cpu().double() * s
    assert ((v - want).abs() <= torch.maximum(v.abs() * 2.0 ** -4, s * 2.0 ** -10) * (1 + 2.0 ** -20) + off).all()


SIZES = [(1, 2, 32), (1, 128, 64), (1, 300, 2048), (3, 129, 95), (7, 64, 1153), (8, 1000, 512), (9, 130, 4000), (16, 256, 1024),
         (17, 384, 300), (33, 128, 640), (64, 514, 1000), (65, 1157, 1153), (100, 640, 256), (129, 300, 2080), (200, 130, 96), (300, 770, 520),
         (520, 258, 1056), (2600, 2570, 800), (513, 255, 129), (700, 129, 5000), (700, 5000, 520), (5000, 5001, 300), (150, 18944, 200), (1, 40000, 130), (40, 20000, 257), (31, 258, 20000)]


@pytest.mark.parametrize("M, N, K", SIZES)
def test_linear(cuda, M, N, K):
    from vila_b200 import ops
    q, w = weight(M, N, K, cuda, spread=1.0)
    a, x = rows8(rand(7, M, K) * torch.exp(rand(8, 1, K)), cuda)
    bias = rand(9, N).to(BF)
    check_product(ops.fp8_linear(a, q), x, w, None)
    check_product(ops.fp8_linear(a, q, bias.to(cuda)), x, w, bias)
    check_rows8(ops.fp8_linear(a, q, bias.to(cuda), to8=True), x, w, bias)


@pytest.mark.parametrize("M", [1, 20, 70, 300, 1100])
@pytest.mark.parametrize("act", ["silu", "relu2", "gelu_tanh", "gelu_erf", "xielu", "swiglu", "geglu", "glu_clamp"])
def test_activations(cuda, M, act, N=770):
    from vila_b200 import ops
    q, w = weight(20, N, 320, cuda)
    a, x = rows8(2 * rand(21, M, 320), cuda)
    bias = rand(22, N).to(BF)
    check_product(ops.fp8_linear(a, q, bias.to(cuda), **act_args(act)), x, w, bias, act)
    check_rows8(ops.fp8_linear(a, q, bias.to(cuda), to8=True, **act_args(act)), x, w, bias, act)


@pytest.mark.parametrize("act", ["none", "silu", "relu2", "gelu_tanh", "gelu_erf", "xielu", "swiglu", "geglu", "glu_clamp"])
def test_activations_of_pairs(cuda, act):
    assert by_pairs(2600, 1802)
    test_activations(cuda, 2600, act, 1802)


@pytest.mark.parametrize("act", ["silu", "swiglu"])
@pytest.mark.parametrize("M", [1, 40, 100, 200])
def test_activations_behind_a_cluster(cuda, M, act):
    from vila_b200 import ops
    q, w = weight(24, 258, 5000, cuda)
    a, x = rows8(rand(25, M, 5000), cuda)
    check_product(ops.fp8_linear(a, q, **act_args(act)), x, w, None, act)
    check_rows8(ops.fp8_linear(a, q, to8=True, **act_args(act)), x, w, None, act)


@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("M", [1, 40, 300])
def test_rows_as_they_come(cuda, M, dtype):
    from vila_b200 import ops
    q, w = weight(26, 200, 300, cuda)
    wide = rand(27, M, 311).to(dtype)
    check_product(ops.fp8_linear(wide.to(cuda)[:, 3:303], q), R.values(*R.quantise(wide[:, 3:303])), w, None)


@pytest.mark.parametrize("M, N", [(2, 200), (40, 200), (300, 200), (2, 40000), (700, 5000)])
def test_views(cuda, M, N):
    from vila_b200 import ops
    q, w = weight(30, N, 288, cuda)
    a, x = rows8(rand(31, M, 288), cuda)
    out = torch.full((M, N + 11), 7.0, dtype=BF, device=cuda)
    got = ops.fp8_linear(a, q, out=out[:, 5:5 + N])
    assert got.data_ptr() == out[:, 5:].data_ptr()
    check_product(got, x, w, None)
    assert (out[:, :5] == 7).all() and (out[:, 5 + N:] == 7).all()
    # codes of rows inside wider ones, with numbers beside them that must not count; scales of more rows than there are
    wide = torch.full((M, 320), 448.0).to(E4M3).to(cuda)
    wide[:, 16:304] = a.codes
    scales = torch.full((3, M + 13 - (M + 1) % 4), math.nan, device=cuda)
    scales = scales[:, :scales.shape[1] // 4 * 4].contiguous()
    scales[:, :M] = a.scales.T
    b = ops.Fp8(wide[:, 16:304], scales[:, :M].T, 1)
    assert b._lds >= M and b._ldc == 320
    check_product(ops.fp8_linear(b, q), x, w, None)
    row = torch.full((N, 1), 7.0, dtype=BF, device=cuda)
    check_product(ops.fp8_linear(rows8(rand(31, M, 288)[:1], cuda)[0], q, out=row.T), x[:1], w, None)


@pytest.mark.parametrize("M, N", [(1, 300), (12, 300), (40, 300), (100, 300), (300, 300), (300, 301), (700, 5000)])
def test_scales_over_the_whole_range(cuda, M, N):
    """Blocks of one row whose sizes are 2^40 apart, rows that differ by 2^60; and blocks of zeros under the largest scales."""
    from vila_b200 import ops
    K = 1024
    sizes = torch.tensor([2.0 ** -20, 2.0 ** 20, 1.0, 2.0 ** -5]).repeat_interleave(128).repeat(K // 512)
    block_rows = torch.exp2(torch.arange(N).float() // 128 % 5 * 15 - 30)
    codes, scales = R.quantise(rand(40, N, K) * sizes * block_rows[:, None], 128)
    a_codes, a_scales = R.quantise(rand(41, M, K) / sizes * torch.exp2(torch.arange(M).float() % 41 - 20)[:, None])
    codes[:, 256:384] = 0
    scales[:, 2] = 3e38
    a_codes[:, 640:768] = 0
    a_scales[:, 5] = 3e38
    a_scales[:, 2] = a_scales[:, 2].clamp(max=448.0 * 1e3)
    scales[:, 5] = scales[:, 5].clamp(max=448.0 * 1e3)
    q, a = ops.fp8_pack(codes.to(E4M3).to(cuda), scales.to(cuda)), ops.fp8_pack(a_codes.to(E4M3).to(cuda), a_scales.to(cuda), block_rows=1)
    check_product(ops.fp8_linear(a, q), R.values(a_codes, a_scales), R.values(codes, scales, 128), None)


@pytest.mark.parametrize("to8", [False, True])
@pytest.mark.parametrize("M, N, K", [(1, 300, 700), (40, 300, 700), (300, 300, 700), (2, 300, 9000), (700, 5000, 700)])
def test_nan_blocks(cuda, M, N, K, to8):
    """A row with an infinity reads as NaN, as does a weight row's output with a NaN code (in 8 bits: its block); nothing else does."""
    from vila_b200 import ops
    x, w = rand(50, M, K), rand(51, N, K) / math.sqrt(K)
    x[M // 2, K - 1] = math.inf
    codes, scales = R.quantise(w, 128)
    codes[N // 3, 5] = math.nan
    q = ops.fp8_pack(codes.to(E4M3).to(cuda), scales.to(cuda))
    a = ops.fp8_quantize(x.to(cuda))
    got = ops.fp8_linear(a, q, to8=to8)
    bad = (ops.fp8_dequantize(got, out_dtype=torch.float32) if to8 else got).isnan().cpu()
    want = torch.zeros(M, N, dtype=torch.bool)
    want[M // 2] = True
    want[:, N // 3] = True
    if to8:
        want[:, N // 3 // 128 * 128:N // 3 // 128 * 128 + 128] = True
    assert torch.equal(bad, want)


def test_sizes_of_nothing_and_gates_of_odd_rows(cuda):
    from vila_b200 import ops
    q, _ = weight(60, 65, 64, cuda)
    none = ops.fp8_quantize(torch.empty(0, 64, device=cuda))
    assert ops.fp8_linear(none, q).shape == (0, 65) and ops.fp8_linear(none, q, to8=True).shape == (0, 65)
    a = ops.fp8_quantize(rand(61, 3, 64).to(cuda))
    with pytest.raises(RuntimeError, match="even number of weight rows"):
        ops.fp8_linear(a, q, swiglu=True)


def test_refusals(cuda):
    from vila_b200 import _lib, ops
    q, _ = weight(62, 64, 64, cuda)
    x = rand(63, 3, 64).to(cuda)
    a = ops.fp8_quantize(x)
    for call, text in ((lambda: ops.fp8_linear(a, ops.fp8_quantize(rand(1, 64, 65).to(cuda), block_rows=128)), "do not fit"),
                       (lambda: ops.fp8_linear(q, q), "a must be Fp8 rows"), (lambda: ops.fp8_linear(a, a), "a must be Fp8 rows"),
                       (lambda: ops.fp8_linear(a, q, rand(1, 64).to(cuda)), "bias must be torch.bfloat16"),
                       (lambda: ops.fp8_linear(a, q, rand(1, 63).to(BF).to(cuda)), "bias must be contiguous"),
                       (lambda: ops.fp8_linear(a, q, act=ops.ACT_SOFTCAP), "unknown activation"),
                       (lambda: ops.fp8_linear(a, q, act=ops.ACT_XIELU), "takes act_params"),
                       (lambda: ops.fp8_linear(a, q, swiglu=True, geglu=True), "one gated unit"),
                       (lambda: ops.fp8_linear(a, q, swiglu=True, act=ops.ACT_SILU), "no other activation"),
                       (lambda: ops.fp8_linear(a, q, out=torch.empty(3, 63, dtype=BF, device=cuda)), "out must be"),
                       (lambda: ops.fp8_linear(a, q, out=torch.empty(3, 64, device=cuda)), "out must be torch.bfloat16"),
                       (lambda: ops.fp8_linear(a, q, to8=True, out=torch.empty(3, 64, dtype=BF, device=cuda)), "takes no out"),
                       (lambda: ops.fp8_quantize(x, block_rows=64), "1 or 128"), (lambda: ops.fp8_quantize(x.half()), "bfloat16 or float32"),
                       (lambda: ops.fp8_quantize(x.T), "consecutive columns"), (lambda: ops.fp8_quantize(x[:, :0]), "consecutive columns"),
                       (lambda: ops.fp8_rmsnorm(x, rand(1, 63).to(cuda), 1e-6), "w must be"),
                       (lambda: ops.fp8_rmsnorm(x, None, 1e-6, residual=x[:2]), "residual must be"),
                       (lambda: ops.fp8_rmsnorm(x, None, 1e-6, out=x), "goes with a residual"),
                       (lambda: ops.fp8_rmsnorm(x, None, 1e-6, residual=x, out=x.to(BF)), "out must be"),
                       (lambda: ops.fp8_rmsnorm(x, None, -1.0), "eps="),
                       (lambda: ops.fp8_rmsnorm(x, None, math.nan), "eps="),
                       (lambda: ops.fp8_rmsnorm(x[:1].expand(3, 64), None, 1e-6, residual=x, out=x[:1].expand(3, 64)), "ld_sum=0"),
                       (lambda: ops.fp8_rmsnorm(torch.zeros(1, 32769, device=cuda), None, 1e-6), "at most 32768"),
                       (lambda: ops.fp8_dequantize(a, out_dtype=torch.float16), "bfloat16 or float32")):
        with pytest.raises(RuntimeError, match=text):
            call()
    # the C entries: null pointers, pointers off their boundaries, strides that do not hold a row
    lib = _lib.load()
    codes, scales = a._ptrs()
    good = (x.data_ptr(), 1, 64, codes, 64, scales, 4, 3, 64, 1)
    for at, bad in ((0, None), (0, x.data_ptr() + 2), (1, 5), (3, None), (3, codes + 8), (4, 56), (4, 48), (5, None), (5, scales + 4), (6, 2), (6, 6), (7, -1), (8, 0), (9, 2)):
        args = list(good)
        args[at] = bad
        assert lib.vila_fp8_quantize(*args, None) == 1, (at, bad)
    w_codes, w_scales = q._ptrs()
    out = torch.full((3, 64), 7.0, dtype=BF, device=cuda)
    fields = dict(a_codes=codes, lda=64, a_scales=scales, ld_as=4, w_codes=w_codes, ldw=64, w_scales=w_scales, ld_ws=1, out=out.data_ptr(), ldo=64, M=3, N=64, K=64)
    for name, bad in (("a_codes", None), ("a_codes", codes + 8), ("lda", 72), ("lda", 48), ("a_scales", None), ("a_scales", scales + 4), ("ld_as", 3), ("ld_as", 0),
                      ("w_codes", None), ("w_codes", w_codes + 1), ("ldw", 65), ("w_scales", w_scales + 2), ("ld_ws", 0), ("out", None), ("out", out.data_ptr() + 1),
                      ("ldo", 63), ("N", 0), ("K", -1), ("M", -1), ("flags", 16), ("bias", out.data_ptr() + 1), ("o_codes", codes)):
        p = _lib.Fp8LinearParams(**{**fields, name: bad})
        assert lib.vila_fp8_linear(C.byref(p), None) == 1, (name, bad)
    p = _lib.Fp8LinearParams(**{**fields, "out": None, "o_codes": codes, "ld_oc": 64, "o_scales": scales, "ld_os": 4})
    if lib.vila_fp8_linear_scratch(C.byref(p)):
        assert lib.vila_fp8_linear(C.byref(p), None) == 1      # no workspace
    torch.cuda.synchronize()
    assert (out == 7).all()


def test_offsets_past_32_bits(cuda):
    """2^31 bytes of codes and more, as rows and as a weight.  Numbers are +-448, their scales 1, so that every sum is a multiple of 448^2 and exact in
    fp32 in whatever order: what lies at the end is what it is by itself, bit by bit."""
    from vila_b200 import ops
    rows, cols, tail = 66048, 33000, 300
    x = torch.empty(rows, cols, dtype=BF, device=cuda)
    for i in range(0, rows, 8192):
        x[i:i + 8192] = torch.randint(0, 2, x[i:i + 8192].shape, dtype=torch.int8, device=cuda)
    x.mul_(2).sub_(1).mul_(448)
    end = x[-tail:].clone()
    q, w = ops.fp8_quantize(x), ops.fp8_quantize(x, block_rows=128)
    assert q.codes.numel() > 1 << 31 and (q.scales == 1).all() and (w.scales == 1).all()
    assert torch.equal(q.codes[-tail:].to(BF), end) and torch.equal(w.codes[-tail:].to(BF), end)
    assert torch.equal(ops.fp8_dequantize(q)[-tail:], end)
    few = ops.fp8_quantize(x[:640].clone(), block_rows=128)
    a = ops.fp8_quantize(end)
    assert torch.equal(ops.fp8_linear(q, few)[-tail:], ops.fp8_linear(a, few))
    w_end = ops.fp8_quantize(x[-512:].clone(), block_rows=128)
    for M in (1, 40, 300):
        b = ops.fp8_quantize(x[:M].clone())
        assert torch.equal(ops.fp8_linear(b, w)[:, -512:], ops.fp8_linear(b, w_end))
    _, total = ops.fp8_rmsnorm(x[:, :32768], None, 1e-6, residual=x[:, :32768])
    assert torch.equal(total[-tail:], 2 * end[:, :32768])


# ---- streams, graphs, waits that run out ---------------------------------------------------------------------
KERNELS = [(1, 300, 700), (1, 300, 9000), (20, 300, 700), (40, 300, 700), (100, 300, 9000), (300, 770, 520), (1500, 1300, 800), (2000, 2400, 800)]


def by_pairs(M, N):
    """whether CTA pairs take it, on 148 SMs"""
    return M > 128 and 4 * -(-(-(-M // 256) * -(-N // 256)) // 74) < 3 * -(-(-(-M // 128) * -(-N // 128)) // 148)


def test_four_streams_at_once(cuda):
    from vila_b200 import ops
    jobs = []
    for i, (M, N, K) in enumerate(KERNELS):
        q, w = weight(70 + i, N, K, cuda)
        a, x = rows8(rand(80 + i, M, K), cuda)
        jobs.append((a, q, ops.fp8_linear(a, q), ops.fp8_linear(a, q, to8=True)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = []
    for r in range(3):
        for i, (a, q, *_) in enumerate(jobs):
            with torch.cuda.stream(streams[(i + r) % 4]):
                got.append((i, ops.fp8_linear(a, q), ops.fp8_linear(a, q, to8=True)))
    torch.cuda.synchronize()
    for i, y, y8 in got:
        assert torch.equal(y, jobs[i][2]) and torch.equal(y8.codes.float(), jobs[i][3].codes.float()) and torch.equal(y8.scales, jobs[i][3].scales)


@pytest.mark.parametrize("M", [1, 40, 300, 1500])
def test_captured_layer(cuda, M):
    """norm, gate / up with a result in 8 bits, down: captured twice, replayed in turn on new rows"""
    from vila_b200 import ops
    gu, down = weight(90, 512, 384, cuda)[0], weight(92, 384, 256, cuda)[0]
    w = rand(93, 384).to(BF).to(cuda)
    x, r = torch.zeros(M, 384, dtype=BF, device=cuda), torch.zeros(M, 384, dtype=BF, device=cuda)

    def layer():
        h, s = ops.fp8_rmsnorm(x, w, 1e-6, residual=r)
        return ops.fp8_linear(ops.fp8_linear(h, gu, swiglu=True, to8=True), down), s

    layer()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            graphs.append((g, layer()))
    for i in range(4):
        x.copy_(rand(94 + i, M, 384).to(BF))
        r.copy_(rand(104 + i, M, 384).to(BF))
        want = layer()
        g, got = graphs[i % 2]
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("tries", [0, 1, -2, -3, -4, -5])
@pytest.mark.parametrize("M, N, K", KERNELS)
def test_waits_that_run_out(cuda, monkeypatch, M, N, K, tries):
    """The launch ends, the next status says so once, and the call after that is right."""
    from vila_b200 import _lib, ops
    w = ops.fp8_quantize(rand(1, N, K).to(cuda), block_rows=128)
    a = ops.fp8_quantize(rand(2, M, K).to(cuda))
    want = ops.fp8_linear(a, w)
    torch.cuda.synchronize()
    ops.check_waits()
    lib = _lib.load()
    with monkeypatch.context() as m:
        m.setattr(lib, "vila_fp8_linear", lambda p, stream: lib.vila_fp8_linear_tries(p, tries, stream))
        out = ops.fp8_linear(a, w)
        torch.cuda.synchronize()
    if tries == 0 or (tries < 0 and (tries != -4 or not by_pairs(M, N))) or not torch.equal(out, want):
        with pytest.raises(RuntimeError, match="ran out of tries"):
            ops.check_waits()
    else:
        try:      # a warp may have given up behind the last wait that its output needs
            ops.check_waits()
        except RuntimeError:
            pass
    ops.check_waits()
    assert torch.equal(ops.fp8_linear(a, w), want)


@pytest.mark.parametrize("M", [1, 40, 300, 1500])
def test_a_weight_of_codes_that_a_launch_just_wrote(cuda, M):
    """A weight whose codes are another launch's 8-bit rows: the layer behind it reads what that launch wrote."""
    from vila_b200 import ops
    a = ops.fp8_quantize(rand(1, M, 1024).to(cuda))
    xs = [rand(2 + i, 640, 1024).to(cuda) for i in range(2)]
    s = torch.rand(5, 8, device=cuda)
    wants = []
    for x in xs:
        codes = ops.fp8_quantize(x).codes
        torch.cuda.synchronize()
        wants.append(ops.fp8_linear(a, ops.fp8_pack(codes, s)))
    torch.cuda.synchronize()
    for i in range(20):
        got = ops.fp8_linear(a, ops.fp8_pack(ops.fp8_quantize(xs[i % 2]).codes, s))
        assert torch.equal(got, wants[i % 2])


@pytest.mark.parametrize("M", [1, 20, 40])
def test_a_long_launch_before_takes_no_tries(cuda, monkeypatch, M):
    """The launch before lets this one begin and runs for milliseconds: waits are counted from its end."""
    from vila_b200 import _lib, ops
    K = 1 << 24
    long_a, long_w = ops.fp8_quantize(torch.ones(1, K, dtype=BF, device=cuda)), ops.fp8_quantize(torch.ones(8, K, dtype=BF, device=cuda), block_rows=128)
    w, a = ops.fp8_quantize(rand(1, 300, 700).to(cuda), block_rows=128), ops.fp8_quantize(rand(2, M, 700).to(cuda))
    want = ops.fp8_linear(a, w)
    torch.cuda.synchronize()
    ops.check_waits()
    lib = _lib.load()
    ops.fp8_linear(long_a, long_w)
    with monkeypatch.context() as m:
        m.setattr(lib, "vila_fp8_linear", lambda p, stream: lib.vila_fp8_linear_tries(p, 256, stream))
        got = ops.fp8_linear(a, w)
    torch.cuda.synchronize()
    ops.check_waits()
    assert torch.equal(got, want)


@pytest.mark.parametrize("role", [0, 1, 3])
@pytest.mark.parametrize("rank", [0, 1])
@pytest.mark.parametrize("M, N, K", [(2000, 2400, 800), (2000, 2400, 5000), (5000, 5000, 700)])
@pytest.mark.parametrize("to8", [False, True])
def test_one_cta_of_a_pair_gives_up(cuda, monkeypatch, M, N, K, to8, rank, role):
    """One CTA of every pair quits while the other has copies in flight that report to it, or expects copies that the first has not
    asked for: the launch ends, says so, and the calls after it are right."""
    from vila_b200 import _lib, ops
    assert by_pairs(M, N)
    w = ops.fp8_quantize(rand(1, N, K).to(cuda), block_rows=128)
    a = ops.fp8_quantize(rand(2, M, K).to(cuda))
    call = lambda: (lambda y: ops.fp8_dequantize(y) if to8 else y)(ops.fp8_linear(a, w, to8=to8, swiglu=to8))  # noqa: E731
    want = call()
    torch.cuda.synchronize()
    ops.check_waits()
    lib = _lib.load()
    with monkeypatch.context() as m:
        m.setattr(lib, "vila_fp8_linear", lambda p, stream: lib.vila_fp8_linear_tries(p, -2 - (role + 4 * (rank + 1)), stream))
        out = ops.fp8_linear(a, w, to8=to8, swiglu=to8)
        torch.cuda.synchronize()
    if rank == 1 and role == 1:      # no such warp: the second CTA's products
        assert torch.equal(ops.fp8_dequantize(out) if to8 else out, want)
    else:
        with pytest.raises(RuntimeError, match="ran out of tries"):
            ops.check_waits()
    ops.check_waits()
    assert torch.equal(call(), want)


# ---- together, as they are used -----------------------------------------------------------------------------
@pytest.mark.parametrize("M", [1, 12, 40, 300, 1100, 5000])
def test_feed_forward_block(cuda, M):
    """norm with the residual, gate / up with a gated unit and a result in 8 bits, down, the next norm: each step from what the one before gave"""
    from vila_b200 import ops
    gu, gu64 = weight(100, 1024, 384, cuda)
    down, down64 = weight(102, 384, 512, cuda)
    x, r, w = rand(104, M, 384).to(BF).to(cuda), rand(105, M, 384).to(BF).to(cuda), (1 + 0.1 * rand(106, 384)).to(BF).to(cuda)
    h, s = ops.fp8_rmsnorm(x, w, 1e-6, residual=r)
    check_norm(h, s, w, 1e-6)
    h64 = R.values(h.codes.cpu(), h.scales.cpu())
    g = ops.fp8_linear(h, gu, swiglu=True, to8=True)
    check_rows8(g, h64, gu64, None, "swiglu")
    y = ops.fp8_linear(g, down)
    check_product(y, R.values(g.codes.cpu(), g.scales.cpu()), down64, None)
    n, t = ops.fp8_rmsnorm(s, w, 1e-6, residual=y)
    assert torch.equal(t, (s.float() + y.float()).to(BF))
    check_norm(n, t, w, 1e-6)


@pytest.mark.parametrize("M", [0, 1, 12, 60, 700])
@pytest.mark.parametrize("N, keep, K", [(200, 8, 288), (200, 7, 288), (96, 64, 100), (2, 1, 32), (640, 320, 512)])
def test_rows_that_stay_as_they_are(cuda, M, N, keep, K):
    from vila_b200 import ops
    w, x, bias = (rand(1, N, K) / math.sqrt(K)).to(BF), rand(2, M, K).to(BF), rand(3, N).to(BF)
    q = ops.fp8_quantize(w.to(cuda), block_rows=128, keep=keep)
    assert q.shape == (N, K) and q.device == x.to(cuda).device and q.nbytes == q.part.nbytes + keep * K * 2
    both = ops.fp8_dequantize(q, out_dtype=torch.float32).cpu()
    eight = R.quantise(w[:N - keep], 128)
    assert torch.equal(both[N - keep:], w[N - keep:].float()) and torch.equal(both[:N - keep], R.values(*eight, 128).float())
    x8 = R.values(*R.quantise(x))
    out = torch.full((M, N + 5), 7.0, dtype=BF, device=cuda)

    def check(got, bias, act="none"):      # the 8-bit rows read quantised rows, the kept ones the rows themselves
        if M:
            n = N - keep
            cut = n // 2 if act == "swiglu" else n
            check_product(got[:, :cut], x8, both[:n], None if bias is None else bias[:n], act)
            check_product(got[:, cut:], x, both[n:], None if bias is None else bias[n:], act)

    check(ops.fp8_linear(x.to(cuda), q, bias.to(cuda), out=out[:, 2:2 + N]), bias)
    assert (out[:, :2] == 7).all() and (out[:, 2 + N:] == 7).all()
    check(ops.linear_any(x.to(cuda), q, act=ops.ACT_SILU), None, "silu")
    if N % 2 == 0 and keep % 2 == 0:
        check(ops.linear_any(x.to(cuda), q, bias=bias.to(cuda), swiglu=True), bias, "swiglu")
    elif M:
        with pytest.raises(RuntimeError, match="even number of weight rows"):
            ops.linear_any(x.to(cuda), q, swiglu=True)
    if M:
        with pytest.raises(RuntimeError, match="bf16 rows and a bf16 result"):
            ops.fp8_linear(ops.fp8_quantize(x.to(cuda)), q)
    for call in (lambda: q.codes, lambda: q.scales, lambda: ops.fp8_linear(ops.fp8_quantize(w.to(cuda)), q, to8=True)):
        with pytest.raises(RuntimeError, match="kept in bf16"):
            call()
    for bad in (N, N + 1, -1):
        with pytest.raises(RuntimeError, match="not all of them"):
            ops.fp8_quantize(w.to(cuda), block_rows=128, keep=bad)
    with pytest.raises(RuntimeError, match="gives bfloat16"):
        ops.linear_any(x.to(cuda), q, out_dtype=torch.float32)


@pytest.mark.parametrize("arch", ["nusovik", "ludazen", "bivizen", "nibelix", "lufatar"])
def test_language_models_on_8_bit_weights(cuda, arch, monkeypatch):
    """Every linear layer on 8-bit weights that a model runs, prompts, portions and decoded tokens, against float64 on the rows that it was
    given; and captured steps against eager ones.  (Whole models are not compared with a second computation: where two of them differ by one
    bf16 rounding, 2^-8, a number lands on the other side of an e4m3 boundary, 2^-3 away, one time in 16 or so.)"""
    import importlib
    from vila_b200 import ops
    from vila_b200.model.registry import MX4_WEIGHTS, quantize_weights
    from vila_b200.serving import TokenEngine
    T = importlib.import_module(f"tests.test_{arch}_gpu")
    name = "aligned" if "aligned" in T.CONFIGS else next(iter(T.CONFIGS))
    cfg, small = T.build(name, BF, seed=3)
    before = {k: v.clone() for k, v in small.state_dict().items()}
    assert quantize_weights(small, "fp8") is small
    names = MX4_WEIGHTS[type(small).__name__.replace("ForCausalLM", "")]
    held = sum(isinstance(getattr(layer, n, None), ops.Fp8) for layer in small.layers for n in names)
    assert held >= len(small.layers)
    assert all(torch.equal(v, before[k]) for k, v in small.state_dict().items())
    linear_any, seen = ops.linear_any, []
    acts = {ops.ACT_NONE: "none", ops.ACT_SILU: "silu", ops.ACT_RELU2: "relu2", ops.ACT_GELU_TANH: "gelu_tanh", ops.ACT_GELU_ERF: "gelu_erf"}

    def checked(x, w, *, bias=None, act=ops.ACT_NONE, swiglu=False, geglu=False, glu_clamp=None, **more):
        got = linear_any(x, w, bias=bias, act=act, swiglu=swiglu, geglu=geglu, glu_clamp=glu_clamp, **more)
        if isinstance(w, ops.Fp8) and act in acts and glu_clamp is None:      # the others' parameters are not what act64 has
            seen.append(x.shape[0])
            kind = "swiglu" if swiglu else "geglu" if geglu else acts[act]
            n = w.part.rows if isinstance(w, ops.Fp8Kept) else w.rows
            values = ops.fp8_dequantize(w, out_dtype=torch.float32).cpu()
            check_product(got[:, :n // 2 if swiglu or geglu else n], R.values(*R.quantise(x)), values[:n], None if bias is None else bias[:n], kind)
            if n < w.rows:
                check_product(got[:, n:], x, values[n:], None if bias is None else bias[n:], kind)
        return got

    eager, captured = TokenEngine(small, 256, 2, graphs=False), TokenEngine(small, 256, 2)
    toks = T.tokens_for(cfg, 60, 5)
    for entries in ([("a", toks[:40], [0, 39]), ("b", toks[:7], [6])], [("a", toks[40:41], [0]), ("b", toks[7:30], [22])],
                    *[[("a", [toks[41 + i]], [0]), ("b", [toks[30 + i]], [0])] for i in range(4)]):
        got = captured.step(entries)
        with monkeypatch.context() as m:
            m.setattr(ops, "linear_any", checked)
            want = eager.step(entries)
        assert torch.equal(got, want)
    assert {47, 24, 2} <= set(seen)
    assert len(small.generate(toks[:9], max_new_tokens=5)[0]) == 5


def test_load_and_command_line(cuda, tmp_path, capsys):
    from llava.cli import infer
    from tests import test_nusovik_gpu as T
    from vila_b200 import ops
    from vila_b200.model import load_language_model
    cfg, model = T.build("aligned", BF, seed=8)
    model.save_pretrained(tmp_path / "m")
    small = load_language_model(tmp_path / "m", weights="fp8")
    assert isinstance(small.layers[0].sel_in, ops.Fp8)
    prompt = T.tokens_for(cfg, 9, 4)
    text = infer.main(["--model-path", str(tmp_path / "m"), "--token-ids", ",".join(map(str, prompt)), "--max-new-tokens", "5", "--weights", "fp8"])
    assert [int(t) for t in text.split(",")] == small.generate(prompt, max_new_tokens=5)[0]
    assert text in capsys.readouterr().out


# ---- prompts in 8 bits -----------------------------------------------------------------------------------------
def qwen(seed=0, layers=3):
    from vila_b200.model.configuration import Qwen2Config
    from vila_b200.model.qwen2 import Qwen2ForCausalLM
    cfg = Qwen2Config(hidden_size=512, intermediate_size=1104, num_hidden_layers=layers, num_attention_heads=4, num_key_value_heads=2, vocab_size=1000)
    llm = Qwen2ForCausalLM(cfg, device="cuda")
    g = torch.Generator().manual_seed(seed)
    with torch.no_grad():
        for name, p in llm.state_dict().items():
            v = torch.randn(p.shape, generator=g)
            p.copy_(1 + 0.1 * v if "norm" in name else v / math.sqrt(p.shape[-1]))
    return llm


def hidden(llm, emb, parts=None, graphed=False):
    cache = llm.new_cache(emb.shape[0])
    run = llm.prefill_hidden_graphed if graphed else llm.prefill_hidden
    return torch.cat([run(e, cache).clone() for e in (emb.split(parts) if parts else [emb])])


@pytest.mark.parametrize("S", [1, 40, 300, 1100])
def test_prompts_in_8_bits(cuda, S):
    """The hidden states of a prompt are the bf16 path's but for the numbers' rounding: an e4m3 number is off by 2^-4 of itself at most, 3.6 % in
    the mean square for any distribution, both factors of a product 5.1 %, and a sum of products of independent signs as much of its own size.  A
    gated unit's product has both of its factors' and one rounding more, 5.1 sqrt 2 + 3.6 < 11 %.  The residual stream adds such errors up
    with the contributions that they belong to: 15 % of the whole, with what earlier layers' errors make of later ones."""
    llm = qwen()
    emb = rand(3, S, 512).to(BF).to(cuda)
    plain = hidden(llm, emb).float()
    assert llm.prefill_in_fp8() is llm
    got = hidden(llm, emb).float()
    off = ((got - plain).norm() / plain.norm()).item()
    assert 1e-4 < off < 0.15
    assert torch.equal(hidden(llm, emb, graphed=True).float(), got) and torch.equal(hidden(llm, emb, graphed=True).float(), got)
    assert torch.equal(hidden(llm.prefill_in_fp8(False), emb).float(), plain)
    assert torch.equal(hidden(llm, emb, graphed=True).float(), plain)


def test_prompts_in_8_bits_are_the_operators_in_turn(cuda):
    """portions of a prompt, a packed batch and changed weights"""
    from vila_b200 import ops
    llm = qwen().prefill_in_fp8()
    emb = rand(4, 90, 512).to(BF).to(cuda)
    whole = hidden(llm, emb).float()
    parted = hidden(llm, emb, parts=40).float()      # rows are quantised one by one: only sums' order and the attention's tiles differ
    assert ((parted - whole).norm() / whole.norm()).item() < 0.02
    # two sequences of a packed row
    logits = llm.forward_packed(emb[None], torch.ones(1, 90, device=cuda), torch.cat([torch.arange(50), torch.arange(40)])[None], torch.tensor([50, 40]))
    for a, b in ((0, 50), (50, 90)):
        want = llm.logits_from_hidden(hidden(llm, emb[a:b])).float()
        assert ((logits[0, a:b].float() - want).norm() / want.norm()).item() < 0.02
    # weights changed in place, as a checkpoint's are copied in: captured prompts are not replayed on the former ones
    before = hidden(llm, emb, graphed=True).clone()
    other = qwen(seed=1)
    with torch.no_grad():
        for p, q in zip(llm.state_dict().values(), other.state_dict().values()):
            p.copy_(q)
    want = hidden(other.prefill_in_fp8(), emb)
    assert torch.equal(hidden(llm, emb, graphed=True), want) and torch.equal(hidden(llm, emb), want) and not torch.equal(want, before)
    ids = llm.generate(inputs_embeds=emb[None], max_new_tokens=4, eos_token_id=None)
    assert ids.shape == (1, 4)
    x = emb.clone()
    layer, eights = llm.model.layers[0], llm._fp8_weights()[0]
    h, x = ops.fp8_rmsnorm(x, layer.input_layernorm.weight, llm.config.rms_norm_eps)
    check_product(ops.fp8_linear(h, eights[0], layer._qkv_b), R.values(h.codes.cpu(), h.scales.cpu()), R.values(*(t.cpu() for t in (eights[0].codes, eights[0].scales)), 128), layer._qkv_b)


def test_weights_that_come_to_lie_where_others_were(cuda):
    """Other tensors at the former ones' addresses, of the same version, are not taken for them."""
    llm, emb = qwen(layers=1).prefill_in_fp8(), rand(4, 90, 512).to(BF).to(cuda)
    layer = llm.model.layers[0]
    first = hidden(llm, emb)
    for i in range(4):
        v = rand(50 + i, 512, 1104).to(BF).to(cuda) / 32
        layer.mlp.down_proj.weight = None      # freed, if nothing else holds it
        layer.mlp.down_proj.weight = torch.nn.Parameter(v.clone(), requires_grad=False)
        got = hidden(llm, emb)
        want = hidden(llm.prefill_in_fp8(), emb)      # quantised anew
        assert torch.equal(got, want) and not torch.equal(got, first)
        first = got


def test_captured_prompts_keep_the_8_bit_weights(cuda):
    """A caller's own capture: refused where the weights would be made in it; behind a change the graph reads the new ones."""
    llm, other, emb = qwen(layers=2).prefill_in_fp8(), qwen(seed=1, layers=2), rand(4, 90, 512).to(BF).to(cuda)
    cache = llm.new_cache(90)
    g = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="outside of a capture"):
        with torch.cuda.graph(g):
            llm.prefill_hidden(emb, cache)
    torch.cuda.synchronize()
    want = hidden(llm, emb)
    cache, g = llm.new_cache(90), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = llm.prefill_hidden(emb, cache)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    with torch.no_grad():
        for p, q in zip(llm.state_dict().values(), other.state_dict().values()):
            p.copy_(q)
    want = hidden(llm, emb)
    junk = [torch.full((1 << 20,), 0x7f, dtype=torch.uint8, device=cuda) for _ in range(16)]      # over what the change has freed
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want) and len(junk) == 16
    # behind a write that torch does not count: called again
    llm.model.layers[0].mlp.down_proj.weight.data.mul_(2)
    want = hidden(llm.prefill_in_fp8(), emb)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_prompts_in_8_bits_on_two_streams(cuda):
    """The first prompt behind a change makes the weights; one on another stream at once reads them made."""
    llm, other, emb = qwen(layers=2).prefill_in_fp8(), qwen(seed=1, layers=2).prefill_in_fp8(), rand(4, 300, 512).to(BF).to(cuda)
    want = hidden(other, emb)
    hidden(llm, emb)
    with torch.no_grad():
        for p, q in zip(llm.state_dict().values(), other.state_dict().values()):
            p.copy_(q)
    torch.cuda.synchronize()
    got = []
    for _ in range(2):
        with torch.cuda.stream(torch.cuda.Stream()):
            got.append(hidden(llm, emb))
    torch.cuda.synchronize()
    assert torch.equal(got[0], want) and torch.equal(got[1], want)


def test_weights_in_one_form_are_not_put_into_the_other(cuda):
    from vila_b200.model import quantize_weights
    import importlib
    T = importlib.import_module("tests.test_nibelix_gpu")
    _, model = T.build(next(iter(T.CONFIGS)), BF, seed=3)
    quantize_weights(model, to="fp8")
    quantize_weights(model, to="fp8")
    with pytest.raises(ValueError, match="held in 8 bits already"):
        quantize_weights(model, to="mx4")
