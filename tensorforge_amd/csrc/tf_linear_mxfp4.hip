// Decode projections by 4-bit weights: y = x . W^T for at most 64 rows, W in
// e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives) with a power-of-two
// scale (e8m0) for each 32 columns of K.
//   y[r][n] = sum_k x[r][k] * e2m1(code[n][k]) * 2^(scale[n][k / 32] - 127)
// in fp32, rounded once; with a residual, round(round(sum) + residual).
#include "tf_common.hpp"

namespace tf {
namespace {

constexpr int32_t kMaxRows = 64;

__device__ __forceinline__ float e2m1(uint32_t code) {
  const float size = code & 4 ? (code & 2 ? (code & 1 ? 6.f : 4.f) : (code & 1 ? 3.f : 2.f))
                              : (code & 2 ? (code & 1 ? 1.5f : 1.f) : (code & 1 ? 0.5f : 0.f));
  return code & 8 ? -size : size;
}

// One wavefront per (column, row), lanes across K.
template <typename T>
__global__ void __launch_bounds__(64)
linear_mxfp4_kernel(const T *__restrict__ x, int64_t x_stride, const uint8_t *__restrict__ weight,
                    int64_t weight_stride, const uint8_t *__restrict__ scales, int64_t scale_stride,
                    const T *__restrict__ residual, int64_t residual_stride, T *__restrict__ y, int64_t y_stride,
                    int32_t k) {
  const int64_t n = blockIdx.x;
  const int64_t r = blockIdx.y;
  float sum = 0.f;
  for (int32_t i = threadIdx.x; i < k; i += 64) {
    const uint32_t code = weight[n * weight_stride + i / 2] >> (4 * (i & 1)) & 15;
    sum += to_float(x[r * x_stride + i]) * ldexpf(e2m1(code), static_cast<int32_t>(scales[n * scale_stride + i / 32]) - 127);
  }
  sum = wave_sum(sum);
  if (threadIdx.x != 0) return;
  T out = from_float<T>(sum);
  if (residual) out = from_float<T>(to_float(out) + to_float(residual[r * residual_stride + n]));
  y[r * y_stride + n] = out;
}

}  // namespace
}  // namespace tf

extern "C" int32_t tf_linear_mxfp4(const void *x, int64_t x_row_stride, const void *weight, int64_t weight_row_stride,
                                   const void *scales, int64_t scale_row_stride, const void *residual,
                                   int64_t residual_row_stride, void *y, int64_t y_row_stride, int32_t m, int32_t n,
                                   int32_t k, int32_t dtype, void *stream) {
  using namespace tf;
  clear_error();
  if (dtype != TF_DTYPE_FLOAT16 && dtype != TF_DTYPE_BFLOAT16)
    return fail(TF_ERROR_UNSUPPORTED, "linear_mxfp4 takes fp16 or bf16 activations");
  if (m < 0 || m > kMaxRows || n < 0 || k <= 0 || k % 32 != 0)
    return fail(TF_ERROR_INVALID_ARGUMENT, "linear_mxfp4 takes at most 64 rows and a K that is a multiple of 32");
  if (m == 0 || n == 0) return TF_SUCCESS;
  if (!x || !weight || !scales || !y) return fail(TF_ERROR_INVALID_ARGUMENT, "null tensor pointer");
  if (x_row_stride < k || weight_row_stride < k / 2 || scale_row_stride < k / 32 || y_row_stride < n ||
      (residual && residual_row_stride < n))
    return fail(TF_ERROR_INVALID_ARGUMENT, "row stride is shorter than the rows");
  if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(weight)) % 16 != 0 || x_row_stride % 8 != 0 ||
      weight_row_stride % 16 != 0)
    return fail(TF_ERROR_INVALID_ARGUMENT, "x and weight rows must be 16-byte aligned");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 grid(n, m);
  if (dtype == TF_DTYPE_FLOAT16)
    hipLaunchKernelGGL((linear_mxfp4_kernel<_Float16>), grid, dim3(64), 0, s, static_cast<const _Float16 *>(x),
                       x_row_stride, static_cast<const uint8_t *>(weight), weight_row_stride,
                       static_cast<const uint8_t *>(scales), scale_row_stride,
                       static_cast<const _Float16 *>(residual), residual_row_stride, static_cast<_Float16 *>(y),
                       y_row_stride, k);
  else
    hipLaunchKernelGGL((linear_mxfp4_kernel<__bf16>), grid, dim3(64), 0, s, static_cast<const __bf16 *>(x),
                       x_row_stride, static_cast<const uint8_t *>(weight), weight_row_stride,
                       static_cast<const uint8_t *>(scales), scale_row_stride, static_cast<const __bf16 *>(residual),
                       residual_row_stride, static_cast<__bf16 *>(y), y_row_stride, k);
  return check_launch("linear_mxfp4");
}
