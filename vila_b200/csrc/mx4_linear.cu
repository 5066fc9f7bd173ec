// vila_mx4_linear: checks of the arguments and the choice of the kernel.
#include "../../include/vila_b200.h"
#include "common.cuh"
#include "glinear_epi.cuh"
#include "kernels.h"
#include "mx4.cuh"

namespace vb {
namespace {
bool on16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
constexpr int kFew = 16;      // rows
// bf16 rows that are cut into 4-bit rows (mx4_tc.cu).  Small layers of up to 8 rows are faster in one launch (mx4_rows.cu), us against us: one row
// of 2048 x 2048 5.5 and 7.6, of 3584 x 3584 7.3 and 8.3, of 8192 x 4096 13.7 and 9.7; 4 rows of 3584 x 3584 7.7 and 8.7, 16 rows
// 12.7 and 10.5.  More than 16 rows are unpacked weights' (mx4_mixed_tc.cu) from about two tiles of 8 rows x 128 weight rows an SM on, us
// against us of those: 17 rows of 3584 x 3584 (84 tiles) 9.9 and 18.3, 64 of 4608 x 3584 (288) 16.4 and 19.1, 17 of 18944 x 3584 (444)
// 20.8 and 19.0, 279 of 1152 x 4304 (315) 31.2 and 21.5.
bool by_pieces(const vila_mx4_linear_params& p) {
  if (p.x == nullptr) return false;
  if (p.M <= kFew) return p.M > 8 || static_cast<long long>(p.N) * p.K > (16ll << 20);
  return static_cast<long long>((p.N + 127) / 128) * ((p.M + 7) / 8) <= 2ll * num_sms();
}
int padded(int K) { return (K + 7) & ~7; }

// rows off 16-byte boundaries -> rows of padded(K) elements; a thread moves 8
__global__ void __launch_bounds__(256) align_kernel(const uint16_t* x, int64_t ldx, uint16_t* out, int M, int K) {
  const int groups = (K + 7) / 8;
  const long long items = static_cast<long long>(M) * groups, step = static_cast<long long>(gridDim.x) * 256;
  for (long long it = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; it < items; it += step) {
    const int m = static_cast<int>(it / groups), k = static_cast<int>(it - static_cast<long long>(m) * groups) * 8;
    const uint16_t* row = x + static_cast<size_t>(m) * ldx + k;
    uint32_t e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = k + i < K ? __ldg(row + i) : 0u;
    stg_v4(out + static_cast<size_t>(m) * groups * 8 + k, make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16));
  }
}
}  // namespace

size_t mx4_linear_scratch(const vila_mx4_linear_params& p) {
  if (p.M <= 0 || p.K <= 0 || p.x == nullptr) return 0;
  if (by_pieces(p)) return mx4_pieces_bytes(p.M, p.K);
  return p.M <= kFew || mx4_mixed_tc_takes(p) ? 0 : static_cast<size_t>(p.M) * padded(p.K) * 2;
}

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
  VB_CHECK(reinterpret_cast<uintptr_t>(p.x) % 2 == 0 && reinterpret_cast<uintptr_t>(p.out) % 2 == 0 && reinterpret_cast<uintptr_t>(p.bias) % 2 == 0,
           "mx4_linear: x, out or bias off its elements' boundaries");
  VB_CHECK(p.M == 1 || p.ldo >= (gated ? p.N / 2 : p.N), "mx4_linear: ldo=%lld N=%d", static_cast<long long>(p.ldo), p.N);
  vila_glinear_ext ext = {};
  ext.act_alpha = p.act_alpha;
  ext.act_limit = p.act_limit;
  ext.act_pos = p.act_pos;
  ext.act_neg = p.act_neg;
  if (p.a_codes != nullptr) return mx4_tc(p, ext, tries, stream);
  if (const size_t want = mx4_linear_scratch(p); want > 0 && p.scratch != nullptr) {
    VB_CHECK(on16(p.scratch) && p.scratch_bytes >= static_cast<int64_t>(want), "mx4_linear: %lld bytes of scratch, %lld wanted, on a 16-byte boundary",
             static_cast<long long>(p.scratch_bytes), static_cast<long long>(want));
    if (by_pieces(p)) return mx4_pieces(p, ext, tries, stream);
    vila_mx4_linear_params q = p;
    q.x = p.scratch;
    q.ldx = padded(p.K);
    const long long blocks = (static_cast<long long>(p.M) * (padded(p.K) / 8) + 255) / 256, most = 16ll * num_sms();
    VB_CUDA(launch_serial(align_kernel, dim3(static_cast<unsigned>(blocks < most ? blocks : most)), dim3(256), 0, stream, static_cast<const uint16_t*>(p.x), p.ldx,
                          static_cast<uint16_t*>(p.scratch), p.M, p.K));
    return mx4_mixed_tc(q, ext, tries, stream);
  }
  if (p.M > kFew && mx4_mixed_tc_takes(p)) return mx4_mixed_tc(p, ext, tries, stream);
  return mx4_rows(p, ext, stream);
}

}  // namespace vb
