// Products with 4-bit weights and group scales:
//   y[r, n] = sum_g s[e, n, g] * sum_{c in g} (q[e, n, c] - z[e, n, g]) * x[r, c]
// One wave a weight row and route: the lanes stride over the row's bytes.
#include "kernels.h"

namespace ktmi {

namespace {

template <typename ST>
__device__ __forceinline__ float scale_at(const void* s, int64_t i) { return (float)((const ST*)s)[i]; }

template <typename T, typename ST>
__global__ __launch_bounds__(256) void w4_rows_kernel(W4Args a) {
  const int lane = threadIdx.x & 63;
  const int64_t r = blockIdx.x;
  int e = 0;
  int64_t xr = r;
  if (a.ids) {
    e = a.ids[r];
    xr = r / a.top_k;
  } else if (a.offsets) {
    e = -1;
    for (int i = 0; i < a.n_experts && e < 0; ++i)
      if (r < a.offsets[i + 1] && r >= a.offsets[i]) e = i;
  }
  for (int64_t n = (int64_t)blockIdx.y * 4 + (threadIdx.x >> 6); n < a.rows; n += (int64_t)gridDim.y * 4) {
    float acc = 0.0f;
    if (e >= 0 && e < a.n_experts) {
      const int64_t row = e * a.rows + n, half = (a.cols + 1) / 2, groups = (a.cols + a.group - 1) / a.group;
      const uint8_t* q = a.codes + row * half;
      const T* x = (const T*)a.x + xr * a.x_stride;
      for (int64_t j = lane; j < half; j += 64) {
        const int64_t g = 2 * j / a.group;
        const float s = scale_at<ST>(a.scales, row * groups + g), z = a.zeros ? (float)a.zeros[row * groups + g] : 8.0f;
        float d = ((float)(q[j] & 15) - z) * (float)x[2 * j];
        if (2 * j + 1 < a.cols) d = fmaf((float)(q[j] >> 4) - z, (float)x[2 * j + 1], d);
        acc = fmaf(s, d, acc);
      }
#pragma unroll
      for (int s = 32; s; s >>= 1) acc += __shfl_xor(acc, s);
    }
    if (lane == 0) ((T*)a.y)[r * a.rows + n] = (T)acc;
  }
}

template <typename T>
void launch_t(const W4Args& a, hipStream_t stream) {
  const int64_t quads = (a.rows + 3) / 4;
  const dim3 grid((unsigned)a.n_routes, (unsigned)(quads < 65535 ? quads : 65535));
  switch (a.scale_dtype) {
    case KTMI_F32: w4_rows_kernel<T, float><<<grid, 256, 0, stream>>>(a); break;
    case KTMI_F16: w4_rows_kernel<T, _Float16><<<grid, 256, 0, stream>>>(a); break;
    default: w4_rows_kernel<T, __bf16><<<grid, 256, 0, stream>>>(a); break;
  }
}

}  // namespace

int64_t w4_workspace(int64_t, int64_t, int64_t) { return 0; }

int launch_w4(const W4Args& a, hipStream_t stream) {
  switch (a.x_dtype) {
    case KTMI_F32: launch_t<float>(a, stream); break;
    case KTMI_F16: launch_t<_Float16>(a, stream); break;
    default: launch_t<__bf16>(a, stream); break;
  }
  KTMI_HIP_TRY(hipGetLastError());
  return KTMI_OK;
}

}  // namespace ktmi
