// Decode projections by 4-bit weights: y = x . W^T for at most 64 rows, W in
// e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives) with a power-of-two
// scale (e8m0) for each 32 columns of K.
//   y[r][n] = sum_k x[r][k] * e2m1(code[n][k]) * 2^(scale[n][k / 32] - 127)
// in fp32, rounded once; with a residual, round(round(sum) + residual).
//
// The products run on v_mfma_f32_16x16x32 with 16 weight rows as the A operand
// and 16 rows of x as the B operand.  A lane loads 16 bytes of a weight row,
// one group of 32 columns, so it holds one scale; the four lanes that share a
// row cover 128 columns.  Which 32 of those 128 meet in one instruction does
// not matter as long as x takes the same order: step s multiplies columns
// 8 s .. 8 s + 7 of each lane's group.  v_cvt_scalef32_pk_bf16_fp4 turns two
// codes into bf16 with the scale applied, exactly, so nothing is left to do to
// the sums.
#include "tf_common.hpp"

namespace tf {
namespace {

constexpr int32_t kMaxRows = 64;
constexpr int32_t kChunk = 128;  // columns of K a wavefront takes at a time

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

struct LinearParams {
  const void *x;
  const uint8_t *weight;
  const uint8_t *scales;
  const void *residual;
  void *y;
  int64_t x_stride, weight_stride, scale_stride, residual_stride, y_stride;
  int32_t m, n, k;
};

template <typename T>
struct Operand;

template <>
struct Operand<__bf16> {
  typedef bf16x8 V;
  static __device__ __forceinline__ V decode(uint32_t codes, float scale) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0);
    const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2);
    const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3);
    return V{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
  }
  static __device__ __forceinline__ f32x4 mfma(V a, V b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};

template <>
struct Operand<_Float16> {
  typedef f16x8 V;
  static __device__ __forceinline__ V decode(uint32_t codes, float scale) {
    const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 0);
    const f16x2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 1);
    const f16x2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 2);
    const f16x2 d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 3);
    return V{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
  }
  static __device__ __forceinline__ f32x4 mfma(V a, V b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};

// fp16 x as the sum of two bf16 values (8 + 3 of its 11 bits: exact), for
// weights that fp16 cannot hold.
__device__ __forceinline__ void split(f16x8 x, bf16x8 &high, bf16x8 &low) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    high[j] = static_cast<__bf16>(static_cast<float>(x[j]));
    low[j] = static_cast<__bf16>(static_cast<float>(x[j]) - static_cast<float>(high[j]));
  }
}

// A workgroup computes 16 NT columns of y for all m <= 16 MT rows, its
// wavefronts taking chunks of K in turn (so they read neighbouring bytes of
// the weight rows together); their sums meet in LDS in the wavefronts' order.
template <typename T, int MT, int NT>
__global__ void __launch_bounds__(MT * NT == 1 ? 1024 : 512) linear_mxfp4_kernel(LinearParams p) {
  typedef typename Operand<T>::V V;
  extern __shared__ f32x4 sums[];  // [wavefronts][NT * MT][64]
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int waves = blockDim.x >> 6;
  const int col = lane & 15;
  const int quad = lane >> 4;
  const int32_t n0 = blockIdx.x * (16 * NT);
  const uint8_t *weight[NT];
  const uint8_t *scale[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int64_t row = min(n0 + 16 * t + col, p.n - 1);
    weight[t] = p.weight + row * p.weight_stride;
    scale[t] = p.scales + row * p.scale_stride;
  }
  const T *x[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
    x[i] = static_cast<const T *>(p.x) + static_cast<int64_t>(min(16 * i + col, p.m - 1)) * p.x_stride;
  f32x4 acc[NT][MT];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[t][i] = f32x4{0.f, 0.f, 0.f, 0.f};

  for (int32_t base = wave * kChunk; base < p.k; base += waves * kChunk) {
    const int32_t k0 = base + 32 * quad;
    u32x4 codes[NT];
    uint32_t exponent[NT];
    V rows[MT][4];
    if (k0 < p.k) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        codes[t] = load_stream16<u32x4>(weight[t] + k0 / 2);
        exponent[t] = scale[t][k0 / 32];
      }
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int s = 0; s < 4; ++s) rows[i][s] = *reinterpret_cast<const V *>(x[i] + k0 + 8 * s);
    } else {  // columns behind K: zero on both sides, whatever x holds there
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        codes[t] = u32x4{0, 0, 0, 0};
        exponent[t] = 127;
      }
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int s = 0; s < 4; ++s) rows[i][s] = V{0, 0, 0, 0, 0, 0, 0, 0};
    }
    if constexpr (__is_same(T, _Float16)) {
      // 0.5 * 2^-13 is fp16's smallest normal value, 6 * 2^13 below its
      // largest: outside, the weights take bf16's range and x two parts.
      bool wide = false;
#pragma unroll
      for (int t = 0; t < NT; ++t) wide |= exponent[t] - (127 - 13) > 26;
      if (__any(wide)) {
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          bf16x8 a[NT];
#pragma unroll
          for (int t = 0; t < NT; ++t)
            a[t] = Operand<__bf16>::decode(codes[t][s], __builtin_bit_cast(float, exponent[t] << 23));
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            bf16x8 high, low;
            split(rows[i][s], high, low);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              acc[t][i] = Operand<__bf16>::mfma(a[t], high, acc[t][i]);
              acc[t][i] = Operand<__bf16>::mfma(a[t], low, acc[t][i]);
            }
          }
        }
        continue;
      }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const float unit = __builtin_bit_cast(float, exponent[t] << 23);
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const V a = Operand<T>::decode(codes[t][s], unit);
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[t][i] = Operand<T>::mfma(a, rows[i][s], acc[t][i]);
      }
    }
  }

#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int i = 0; i < MT; ++i) sums[(wave * NT * MT + t * MT + i) * 64 + lane] = acc[t][i];
  __syncthreads();
  for (int item = threadIdx.x; item < NT * MT * 64; item += blockDim.x) {
    f32x4 sum = sums[item];
    for (int w = 1; w < waves; ++w) sum += sums[w * NT * MT * 64 + item];
    const int tile = item >> 6;
    const int32_t r = 16 * (tile % MT) + (item & 15);
    const int32_t first = n0 + 16 * (tile / MT) + 4 * ((item >> 4) & 3);
    if (r >= p.m) continue;
    T *out = static_cast<T *>(p.y) + r * p.y_stride;
    const T *residual = p.residual ? static_cast<const T *>(p.residual) + r * p.residual_stride : nullptr;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (first + j >= p.n) break;
      T value = from_float<T>(sum[j]);
      if (residual) value = from_float<T>(to_float(value) + to_float(residual[first + j]));
      out[first + j] = value;
    }
  }
}

template <typename T, int MT, int NT>
int32_t launch_linear(const LinearParams &p, int waves, hipStream_t stream) {
  const size_t lds = static_cast<size_t>(waves) * NT * MT * 64 * sizeof(f32x4);
  if (lds > 65536) {
    static const hipError_t raised = hipFuncSetAttribute(reinterpret_cast<const void *>(&linear_mxfp4_kernel<T, MT, NT>),
                                                         hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
    if (raised != hipSuccess) return fail(TF_ERROR_LAUNCH, "linear_mxfp4: the LDS limit was refused");
  }
  hipLaunchKernelGGL((linear_mxfp4_kernel<T, MT, NT>), dim3((p.n + 16 * NT - 1) / (16 * NT)), dim3(64 * waves),
                     lds, stream, p);
  return check_launch("linear_mxfp4");
}

template <typename T, int MT>
int32_t launch_columns(const LinearParams &p, int tiles, int waves, hipStream_t stream) {
  switch (tiles) {
    case 1: return launch_linear<T, MT, 1>(p, waves, stream);
    case 2: return launch_linear<T, MT, 2>(p, waves, stream);
    default: return launch_linear<T, MT, 4>(p, waves, stream);
  }
}

template <typename T>
int32_t launch_rows(const LinearParams &p, int tiles, int waves, hipStream_t stream) {
  switch ((p.m + 15) / 16) {
    case 1: return launch_columns<T, 1>(p, tiles, waves, stream);
    case 2: return launch_columns<T, 2>(p, tiles, waves, stream);
    case 3: return launch_columns<T, 3>(p, tiles, waves, stream);
    default: return launch_columns<T, 4>(p, tiles, waves, stream);
  }
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
  const LinearParams p{x,           static_cast<const uint8_t *>(weight), static_cast<const uint8_t *>(scales),
                       residual,    y,                                    x_row_stride,
                       weight_row_stride, scale_row_stride,               residual_row_stride,
                       y_row_stride, m,                                   n,
                       k};
  const int32_t chunks = (k + kChunk - 1) / kChunk;
  const int32_t columns = (n + 15) / 16;
  const int tiles = columns >= 1024 ? 4 : columns >= 512 ? 2 : 1;
  const int waves = chunks < 8 ? chunks : 8;
  hipStream_t s = static_cast<hipStream_t>(stream);
  return dtype == TF_DTYPE_FLOAT16 ? launch_rows<_Float16>(p, tiles, waves, s)
                                   : launch_rows<__bf16>(p, tiles, waves, s);
}
