// vila_mx4_linear: checks of the arguments and the choice of the kernel.
#include "../../include/vila_b200.h"
#include "common.cuh"
#include "glinear_epi.cuh"
#include "kernels.h"
#include "mx4.cuh"

namespace vb {
namespace {
bool on16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
}  // namespace

int mx4_linear(const vila_mx4_linear_params& p, cudaStream_t stream, int tries) {
  if (wait_status()) return 1;   // an earlier launch gave up: nothing is built on its output
  VB_CHECK(p.M >= 0 && p.N > 0 && p.K > 0 && p.M <= (1 << 30) && p.N <= (1 << 30) && p.K <= (1 << 30), "mx4_linear: M=%d N=%d K=%d", p.M, p.N, p.K);
  const int gated = p.flags & kGluFlags;
  VB_CHECK((p.flags & ~kGluFlags) == 0 && (gated & (gated - 1)) == 0, "mx4_linear: flags=%d (one gated unit at most)", p.flags);
  VB_CHECK(gated == 0 || p.N % 2 == 0, "mx4_linear: a gated unit has an even number of weight rows (N=%d)", p.N);
  VB_CHECK(gated == 0 || p.act == VILA_ACT_NONE, "mx4_linear: a gated unit takes no other activation (act=%d)", p.act);
  VB_CHECK(p.act == VILA_ACT_NONE || p.act == VILA_ACT_GELU_TANH || p.act == VILA_ACT_GELU_ERF || p.act == VILA_ACT_SILU ||
               p.act == VILA_ACT_RELU2 || p.act == VILA_ACT_XIELU,
           "mx4_linear: unknown activation %d", p.act);
  if (p.M == 0) return 0;
  VB_CHECK((p.x != nullptr) != (p.a_codes != nullptr), "mx4_linear: the rows are bf16 numbers or codes with scales, one of the two");
  VB_CHECK(p.w_codes != nullptr && p.w_scales != nullptr && p.out != nullptr && (p.a_codes == nullptr || p.a_scales != nullptr),
           "mx4_linear: a null pointer");
  VB_CHECK(on16(p.w_codes) && on16(p.w_scales) && on16(p.a_codes) && on16(p.a_scales), "mx4_linear: codes and scales start on 16-byte boundaries");
  VB_CHECK(p.ldo >= (gated ? p.N / 2 : p.N), "mx4_linear: ldo=%lld N=%d", static_cast<long long>(p.ldo), p.N);
  vila_glinear_ext ext = {};
  ext.act_alpha = p.act_alpha;
  ext.act_limit = p.act_limit;
  ext.act_pos = p.act_pos;
  ext.act_neg = p.act_neg;
  if (p.a_codes != nullptr && p.M > 16) return mx4_tc(p, ext, tries, stream);
  if (p.M > 16 && mx4_mixed_tc_takes(p)) return mx4_mixed_tc(p, ext, tries, stream);
  return mx4_rows(p, ext, stream);
}

}  // namespace vb
