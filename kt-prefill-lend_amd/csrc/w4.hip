// Products with 4-bit weights: the choice of kernels (w4_kernel.h, one file for each activation type) and
// the routes' order for calls with more ids than a wave holds.
#include "kernels.h"

namespace ktmi {

namespace {

int launch_any(const W4Args& a, hipStream_t stream, ktmi_w4_kernel* tell) {
  return a.x_dtype == KTMI_F32   ? launch_w4_f32(a, stream, tell)
         : a.x_dtype == KTMI_F16 ? launch_w4_f16(a, stream, tell)
                                 : launch_w4_bf16(a, stream, tell);
}

// workspace of a call with more ids than a wave holds: the routes' order (offsets, perm, pos) and the
// sort's counts
int64_t ints(int64_t n) { return (n + 3) / 4 * 4; }

}  // namespace

int64_t w4_workspace(int64_t tokens, int64_t top_k, int64_t E) {
  const int64_t R = tokens * top_k;
  if (R <= W4_IDS) return 0;
  return 4 * (ints(E + 1) + 2 * ints(R) + ints(moe_sort_counts(tokens, top_k) * (E + 1)));
}

int launch_w4(const W4Args& a, hipStream_t stream, ktmi_w4_kernel* tell) {
  int rc;
  if (a.ids && a.n_routes > W4_IDS && a.cols >= W4_STEP) {
    int* offsets = (int*)a.ws;
    int* perm = offsets + ints(a.n_experts + 1);
    int* pos = perm + ints(a.n_routes);
    rc = tell ? KTMI_OK
              : launch_moe_sort(nullptr, 2, 0, 0, a.ids, a.n_routes / a.top_k, a.top_k, a.n_experts, nullptr, offsets, perm,
                                pos, pos + ints(a.n_routes), stream);
    if (rc) return rc;
    W4Args b = a;
    b.ids = nullptr, b.offsets = offsets, b.perm = perm;
    rc = launch_any(b, stream, tell);
  } else {
    rc = launch_any(a, stream, tell);
  }
  if (rc || tell) return rc;
  KTMI_HIP_TRY(hipGetLastError());
  return KTMI_OK;
}

}  // namespace ktmi
