// vila_fp8_linear: checks of the arguments, rows that are quantised behind the product.
#include "../../include/vila_b200.h"
#include "fp8.cuh"
#include "glinear_epi.cuh"
#include "kernels.h"

namespace vb {
namespace {
bool on(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
int width(const vila_fp8_linear_params& p) { return p.flags & kGluFlags ? p.N / 2 : p.N; }

// The scratch: rows that are quantised here (codes, scales), then an unrounded result, which a launch of its own quantises.
int64_t pitch(int cols) { return (static_cast<int64_t>(cols) + 15) / 16 * 16; }
int64_t lds(int rows) { return (static_cast<int64_t>(rows) + 3) / 4 * 4; }
int64_t rows_bytes(const vila_fp8_linear_params& p) { return p.x == nullptr ? 0 : p.M * pitch(p.K) + fp8_blocks(p.K) * lds(p.M) * 4; }
int64_t result_bytes(const vila_fp8_linear_params& p) { return p.o_codes == nullptr || fp8_pair_takes(p) ? 0 : static_cast<int64_t>(p.M) * width(p) * 4; }
}  // namespace

size_t fp8_linear_scratch(const vila_fp8_linear_params& p) {
  if (p.M <= 0 || p.N <= 0 || p.K <= 0) return 0;
  return static_cast<size_t>(rows_bytes(p) + result_bytes(p));
}

int fp8_linear(const vila_fp8_linear_params& given, cudaStream_t stream, int tries) {
  vila_fp8_linear_params p = given;
  if (wait_status()) return 1;   // an earlier launch gave up: nothing is built on its output
  VB_CHECK(p.M >= 0 && p.N > 0 && p.K > 0 && p.M <= (1 << 30) && p.N <= (1 << 30) && p.K <= (1 << 30), "fp8_linear: M=%d N=%d K=%d", p.M, p.N, p.K);
  const int gated = p.flags & kGluFlags;
  VB_CHECK((p.flags & ~(kGluFlags | VILA_FLAG_STATIC_W)) == 0 && (gated & (gated - 1)) == 0, "fp8_linear: flags=%d (one gated unit at most)", p.flags);
  VB_CHECK(gated == 0 || p.N % 2 == 0, "fp8_linear: a gated unit has an even number of weight rows (N=%d)", p.N);
  VB_CHECK(gated == 0 || p.act == VILA_ACT_NONE, "fp8_linear: a gated unit takes no other activation (act=%d)", p.act);
  VB_CHECK(p.act == VILA_ACT_NONE || p.act == VILA_ACT_GELU_TANH || p.act == VILA_ACT_GELU_ERF || p.act == VILA_ACT_SILU ||
               p.act == VILA_ACT_RELU2 || p.act == VILA_ACT_XIELU,
           "fp8_linear: unknown activation %d", p.act);
  VB_CHECK((p.out != nullptr) != (p.o_codes != nullptr) || p.M == 0, "fp8_linear: a result in bf16, or codes with scales, one of the two");
  if (p.M == 0) return 0;
  const int64_t want = static_cast<int64_t>(fp8_linear_scratch(p));
  VB_CHECK(want == 0 || (p.scratch != nullptr && on(p.scratch, 16) && p.scratch_bytes >= want), "fp8_linear: %lld bytes of scratch, %lld wanted, on a 16-byte boundary",
           static_cast<long long>(p.scratch_bytes), static_cast<long long>(want));
  if (p.x != nullptr) {
    VB_CHECK(p.a_codes == nullptr && p.a_scales == nullptr, "fp8_linear: the rows are numbers or codes with scales, one of the two");
    p.a_codes = p.scratch;
    p.lda = pitch(p.K);
    p.a_scales = reinterpret_cast<const float*>(static_cast<const uint8_t*>(p.scratch) + p.M * p.lda);
    p.ld_as = lds(p.M);
  }
  VB_CHECK(p.a_codes != nullptr && p.a_scales != nullptr && p.w_codes != nullptr && p.w_scales != nullptr, "fp8_linear: a null pointer");
  VB_CHECK(on(p.a_codes, 16) && on(p.w_codes, 16) && p.lda % 16 == 0 && p.ldw % 16 == 0 && p.lda >= p.K && p.ldw >= p.K,
           "fp8_linear: rows of codes start on 16-byte boundaries, lda=%lld ldw=%lld K=%d", static_cast<long long>(p.lda), static_cast<long long>(p.ldw), p.K);
  VB_CHECK(on(p.a_scales, 16) && p.ld_as % 4 == 0 && p.ld_as >= p.M, "fp8_linear: a's scales start on 16-byte boundaries, ld_as=%lld M=%d",
           static_cast<long long>(p.ld_as), p.M);
  VB_CHECK(on(p.w_scales, 4) && p.ld_ws >= fp8_blocks(p.K), "fp8_linear: w's scales: ld_ws=%lld K=%d", static_cast<long long>(p.ld_ws), p.K);
  VB_CHECK(on(p.bias, 2), "fp8_linear: bias off its elements' boundaries");
  vila_glinear_ext ext = {};
  ext.act_alpha = p.act_alpha;
  ext.act_limit = p.act_limit;
  ext.act_pos = p.act_pos;
  ext.act_neg = p.act_neg;
  const int n = width(p);
  if (p.out != nullptr) {
    VB_CHECK(on(p.out, 2) && (p.M == 1 || p.ldo >= n), "fp8_linear: out off its elements' boundaries, or ldo=%lld for %d columns", static_cast<long long>(p.ldo), n);
  } else {
    VB_CHECK(p.o_scales != nullptr && on(p.o_codes, 16) && p.ld_oc % 16 == 0 && p.ld_oc >= n && on(p.o_scales, 16) && p.ld_os % 4 == 0 && p.ld_os >= p.M,
             "fp8_linear: the result's codes and scales start on 16-byte boundaries, ld_oc=%lld ld_os=%lld for %d rows of %d", static_cast<long long>(p.ld_oc),
             static_cast<long long>(p.ld_os), p.M, n);
  }
  if (p.x != nullptr)
    if (int rc = fp8_quantize(p.x, p.x_dtype, p.ldx, const_cast<void*>(p.a_codes), p.lda, const_cast<float*>(p.a_scales), p.ld_as, p.M, p.K, 1, stream)) return rc;
  if (fp8_pair_takes(p)) return fp8_pair(p, ext, tries, stream);
  if (p.out != nullptr) return fp8_tc(p, ext, nullptr, tries, stream);
  float* z = reinterpret_cast<float*>(static_cast<uint8_t*>(p.scratch) + rows_bytes(p));
  if (int rc = fp8_tc(p, ext, z, tries, stream)) return rc;
  return fp8_quantize(z, VILA_DT_F32, n, p.o_codes, p.ld_oc, p.o_scales, p.ld_os, p.M, n, 1, stream);
}

}  // namespace vb
