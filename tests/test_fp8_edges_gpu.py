"""GPU: linear layers on 8-bit rows where launches follow one another closely, and at the ends of their numbers' range."""
import ctypes as C

import pytest
import torch

from tests import fp8_reference as R
from tests.test_fp8_gpu import KERNELS, check_rows8, nothing_left_behind, rand, rows8, weight  # noqa: F401
from tests.test_mx4_gpu import check_product

pytestmark = pytest.mark.gpu
BF, E4M3 = torch.bfloat16, torch.float8_e4m3fn


@pytest.mark.parametrize("rows", ["codes", "bf16"])
@pytest.mark.parametrize("M, N, K", KERNELS)
def test_a_weight_written_in_place_right_before(cuda, M, N, K, rows):
    """The layer reads what the launch before wrote into its weight, whether rows are quantised between the two or not."""
    from vila_b200 import ops
    w, x = ops.fp8_quantize(rand(1, N, K).to(cuda), block_rows=128), rand(2, M, K).to(BF).to(cuda)
    a = x if rows == "bf16" else ops.fp8_quantize(x)
    xs = [rand(3 + i, N, K).to(cuda) for i in range(2)]
    forms = [ops.fp8_quantize(t, block_rows=128) for t in xs]
    torch.cuda.synchronize()
    wants = [ops.fp8_linear(a, q) for q in forms]
    torch.cuda.synchronize()
    assert not torch.equal(*wants) and not w.static_w
    for i in range(20):
        w._held().copy_(forms[i % 2]._held())
        assert torch.equal(ops.fp8_linear(a, w), wants[i % 2])
        assert torch.equal(ops.fp8_linear(a, ops.fp8_quantize(xs[i % 2], block_rows=128)), wants[i % 2])
    w.static_w = True      # behind a synchronisation the same numbers
    torch.cuda.synchronize()
    assert torch.equal(ops.fp8_linear(a, w), wants[1])


def test_a_flag_that_a_layer_does_not_know_is_refused(cuda):
    from vila_b200 import _lib, ops
    (q, _), (a, _) = weight(1, 64, 64, cuda), rows8(rand(2, 3, 64), cuda)
    out = torch.full((3, 64), 7.0, dtype=BF, device=cuda)
    codes, scales = a._ptrs()
    w_codes, w_scales = q._ptrs()
    for flags, ok in ((2, True), (16, False), (18, False), (-1, False), (2 | 1 | 8, False)):
        p = _lib.Fp8LinearParams(a_codes=codes, lda=64, a_scales=scales, ld_as=4, w_codes=w_codes, ldw=64, w_scales=w_scales, ld_ws=1, out=out.data_ptr(), ldo=64,
                                 M=3, N=64, K=64, flags=flags)
        torch.cuda.synchronize()
        assert (_lib.load().vila_fp8_linear(C.byref(p), None) == 0) == ok
    torch.cuda.synchronize()
    assert torch.equal(out, ops.fp8_linear(a, q))


@pytest.mark.parametrize("tries", [0, 1, -2, -3, -4, -5])
@pytest.mark.parametrize("M, N, K", [(1, 300, 9000), (20, 300, 700), (100, 300, 9000), (300, 770, 520)])
def test_waits_that_run_out_with_weights_fetched_ahead(cuda, monkeypatch, M, N, K, tries):
    """What was fetched ahead has landed before the launch ends, whoever gave up; the next status says so once, and the call after that is right."""
    from vila_b200 import _lib, ops
    w, a = ops.fp8_quantize(rand(1, N, K).to(cuda), block_rows=128), ops.fp8_quantize(rand(2, M, K).to(cuda))
    want = ops.fp8_linear(a, w)
    torch.cuda.synchronize()
    w.static_w = True
    ops.check_waits()
    lib = _lib.load()
    with monkeypatch.context() as m:
        m.setattr(lib, "vila_fp8_linear", lambda p, stream: lib.vila_fp8_linear_tries(p, tries, stream))
        out = ops.fp8_linear(a, w)
        torch.cuda.synchronize()
    if tries <= 0 or not torch.equal(out, want):
        with pytest.raises(RuntimeError, match="ran out of tries"):
            ops.check_waits()
    else:
        try:      # a warp may have given up behind the last wait that its output needs
            ops.check_waits()
        except RuntimeError:
            pass
    ops.check_waits()
    assert torch.equal(ops.fp8_linear(a, w), want)


@pytest.mark.parametrize("to8", [False, True])
@pytest.mark.parametrize("M, N, K", KERNELS + [(32, 130, 300), (128, 130, 1300), (129, 300, 700)])
def test_products_of_scales_past_fp32(cuda, M, N, K, to8):
    """Blocks whose scales' product is past fp32's largest number: sums that make it finite again are what they are, sums of zero count nothing, and tokens
    beside them whose product is an ordinary one are what they were."""
    from vila_b200 import ops
    blocks, tiny = -(-K // 128), torch.tensor([0.0, 2.0 ** -9, -2.0 ** -9, 2.0 ** -8])
    pick = torch.Generator().manual_seed(5)
    codes, scales = R.quantise(rand(1, N, K), 128)
    a_codes, a_scales = R.quantise(rand(2, M, K))
    codes[:, 128:256] = tiny[torch.randint(4, (N, 128), generator=pick)].double()
    a_codes[:, 128:256] = tiny[torch.randint(4, (M, 128), generator=pick)].double()
    scales[:, 1] = 1.5 * 2.0 ** 65
    a_scales[:, 1] = torch.where(torch.arange(M) % 3 == 0, 1.25 * 2.0 ** 66, 2.0 ** -20)      # sums up to 128 x 2^-16: 2^123
    a_codes[:, 256:384], a_scales[:, 2] = 0, 3e38
    scales[:, 2] = 3e38
    assert blocks > 2 and (a_scales[0, 1].double() * scales[0, 1].double()) > 3.5e38
    q, a = ops.fp8_pack(codes.to(E4M3).to(cuda), scales.to(cuda)), ops.fp8_pack(a_codes.to(E4M3).to(cuda), a_scales.to(cuda), block_rows=1)
    got, x, w = ops.fp8_linear(a, q, to8=to8), R.values(a_codes, a_scales), R.values(codes, scales, 128)
    (check_rows8 if to8 else check_product)(got, x, w, None)


@pytest.mark.parametrize("M, N, K", KERNELS + [(32, 130, 300), (128, 130, 1300)])
def test_what_fp32_cannot_hold_is_an_infinity(cuda, M, N, K):
    from vila_b200 import ops
    codes, scales = R.quantise(rand(1, N, K), 128)
    a_codes, a_scales = R.quantise(rand(2, M, K))
    plain = ops.fp8_linear(ops.fp8_pack(a_codes.to(E4M3).to(cuda), a_scales.to(cuda), block_rows=1), ops.fp8_pack(codes.to(E4M3).to(cuda), scales.to(cuda)))
    a_codes[:, 128:256] = 0
    base = ops.fp8_linear(ops.fp8_pack(a_codes.to(E4M3).to(cuda), a_scales.to(cuda), block_rows=1), ops.fp8_pack(codes.to(E4M3).to(cuda), scales.to(cuda)))
    m, sign = M // 2, (torch.arange(N) % 3 - 1).double()
    a_codes[m, 133], a_scales[m, 1], scales[:, 1] = 1.0, 3e38, 4.0
    codes[:, 133] = sign
    got = ops.fp8_linear(ops.fp8_pack(a_codes.to(E4M3).to(cuda), a_scales.to(cuda), block_rows=1), ops.fp8_pack(codes.to(E4M3).to(cuda), scales.to(cuda)))
    want = base.clone()
    want[m] = torch.where(sign.to(cuda) == 0, base[m], (sign * torch.inf).to(cuda).to(BF))
    assert torch.equal(got, want) and not torch.equal(plain, base)


def one_term(M, N, K, z, cuda):
    """Rows and a weight whose sum of token m is z[m] times +-1 (columns' turn), exact in fp32: one number each, z a power of two."""
    from vila_b200 import ops
    codes, a_codes = torch.zeros(N, K), torch.zeros(M, K)
    codes[:, K // 2], a_codes[:, K // 2] = torch.where(torch.arange(N) % 2 == 0, 1.0, -1.0), 1.0
    a_scales = torch.full((M, -(-K // 128)), 0.5)
    a_scales[:, K // 2 // 128] = z
    a = ops.fp8_pack(a_codes.to(E4M3).to(cuda), a_scales.to(cuda), block_rows=1)
    return a, ops.fp8_pack(codes.to(E4M3).to(cuda), torch.ones(-(-N // 128), a_scales.shape[1], device=cuda)), torch.outer(z.double(), codes[:, K // 2].double())


@pytest.mark.parametrize("M, N, K", KERNELS)
def test_small_numbers_through_xielu(cuda, M, N, K):
    """z down to -+2^-40.  e^z - 1 - z is a_neg = 0.4 times, and near 0 the result is about z / 2.  Above -1/16 the series leaves out z^5 / 120, 2^-22 of that; from there
    on __expf is off by at most 2 units of 2^-24 and two roundings by half a one each: 3 x 0.4 x 2^-24 of 2^-5 and more, below 2^-18; the sum's own roundings are 2^-23.
    Then half a step of its type: bf16 2^-8, or e4m3's 2^-4 and 2^-10 of its block's scale."""
    from vila_b200 import ops
    z = torch.exp2(-(torch.arange(M) % 41).float())
    a, w, sums = one_term(M, N, K, z, cuda)
    want = torch.where(sums > 0, 0.7 * sums * sums + sums / 2, 0.4 * (torch.expm1(sums) - sums) + sums / 2)
    args = dict(act=ops.ACT_XIELU, act_params=(0.7, 0.4))
    got = ops.fp8_linear(a, w, **args).double().cpu()
    assert ((got - want).abs() <= want.abs() * (2.0 ** -8 + 2.0 ** -18)).all()
    q = ops.fp8_linear(a, w, to8=True, **args)
    v, s = ops.fp8_dequantize(q, out_dtype=torch.float32).double().cpu(), R.per_element(q.scales.cpu(), 1, M, N)
    assert ((v - want).abs() <= torch.maximum(want.abs() * 2.0 ** -4, s * 2.0 ** -10) * (1 + 2.0 ** -16) + want.abs() * 2.0 ** -18).all()


@pytest.mark.parametrize("M, N, K", KERNELS)
def test_far_negative_gates(cuda, M, N, K):
    """silu of -16, -32, -64 and their positive ones, times u = minus the same.  __expf(x) is off by 2 + 1.2 |x| units of 2^-23, the division by 2 more and the products by half
    one each: (5 + 1.2 |x|) 2^-23; then half a step of the result's type."""
    from vila_b200 import ops
    N = N // 4 * 4
    z = torch.exp2(4.0 + torch.arange(M) % 3)
    a, w, sums = one_term(M, N, K, z, cuda)      # gates z, ups -z
    codes = w.codes.clone()
    codes[2::4], codes[3::4] = codes[3::4].clone(), codes[2::4].clone()      # and the other way round
    sums[:, 2::4], sums[:, 3::4] = -sums[:, 2::4], -sums[:, 3::4]
    g, u = sums[:, 0::2], sums[:, 1::2]
    want = g * torch.sigmoid(g) * u
    more = want.abs() * (5 + 1.2 * g.abs()) * 2.0 ** -23
    got = ops.fp8_linear(a, ops.fp8_pack(codes, w.scales), swiglu=True).double().cpu()
    assert (want[0] != 0).all() and ((got - want).abs() <= want.abs() * 2.0 ** -8 * (1 + 2.0 ** -16) + more).all()
    q = ops.fp8_linear(a, ops.fp8_pack(codes, w.scales), swiglu=True, to8=True)
    v, s = ops.fp8_dequantize(q, out_dtype=torch.float32).double().cpu(), R.per_element(q.scales.cpu(), 1, *want.shape)
    assert ((v - want).abs() <= torch.maximum(want.abs() * 2.0 ** -4, s * 2.0 ** -10) * (1 + 2.0 ** -15) + more).all()
