// Log probabilities of given tokens, the entropy of each row's distribution
// and its most likely tokens.
//
// For a row x: m = max x, S = sum exp(x - m);
//   log p(i) = (x[i] - m) - log S
//   H = log S - (sum (x - m) exp(x - m)) / S       (both terms >= 0)
// with the term of x = -inf zero.  The alternatives are ordered by value,
// equal values by index, a NaN above every number (as in tf_argmax_rows).
#include "tf_common.hpp"

namespace tf {
namespace {

constexpr int32_t kMaxTop = 32;
constexpr int kThreads = 256;

// An unsigned integer that orders as the value does: -0 equals +0, NaN last.
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t bits = __builtin_bit_cast(uint32_t, x + 0.f);
  return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}

template <typename F>
__device__ __forceinline__ float block_reduce(float v, float *slots, F combine) {
  for (int offset = 32; offset > 0; offset >>= 1) v = combine(v, __shfl_xor(v, offset, 64));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) slots[threadIdx.x >> 6] = v;
  __syncthreads();
  v = slots[0];
  for (int w = 1; w < kThreads / 64; ++w) v = combine(v, slots[w]);
  return v;
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
token_logprobs_kernel(const T *__restrict__ logits, int64_t row_stride, int32_t columns,
                      const int64_t *__restrict__ tokens, float *__restrict__ logprobs, float *__restrict__ entropy,
                      float *__restrict__ top_logprobs, int64_t *__restrict__ top_tokens, int32_t top_k) {
  __shared__ float slots[kThreads / 64];
  __shared__ unsigned long long keys[kThreads / 64];
  const int64_t r = blockIdx.x;
  const T *row = logits + r * row_stride;
  float m = -__builtin_inff();
  for (int32_t c = threadIdx.x; c < columns; c += kThreads) m = fmaxf(m, to_float(row[c]));
  m = block_reduce(m, slots, [](float a, float b) { return fmaxf(a, b); });
  float sum = 0.f, weighted = 0.f;
  for (int32_t c = threadIdx.x; c < columns; c += kThreads) {
    const float d = to_float(row[c]) - m;
    const float e = expf(d);
    sum += e;
    weighted += e == 0.f ? 0.f : d * e;
  }
  auto add = [](float a, float b) { return a + b; };
  sum = block_reduce(sum, slots, add);
  weighted = block_reduce(weighted, slots, add);
  const float log_sum = logf(sum);
  if (threadIdx.x == 0) {
    const int64_t token = tokens[r];
    logprobs[r] = token >= 0 && token < columns ? (to_float(row[token]) - m) - log_sum : __builtin_nanf("");
    entropy[r] = log_sum - weighted / sum;
  }
  unsigned long long last = ~0ull;
  for (int32_t j = 0; j < top_k; ++j) {
    unsigned long long best = 0;
    for (int32_t c = threadIdx.x; c < columns; c += kThreads) {
      const unsigned long long key =
          static_cast<unsigned long long>(order_key(to_float(row[c]))) << 32 | (0x7fffffffu - c);
      if (key < last && key > best) best = key;
    }
    for (int offset = 32; offset > 0; offset >>= 1) {
      const unsigned long long other = __shfl_xor(best, offset, 64);
      best = other > best ? other : best;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) keys[threadIdx.x >> 6] = best;
    __syncthreads();
    for (int w = 0; w < kThreads / 64; ++w) best = keys[w] > best ? keys[w] : best;
    last = best;
    if (threadIdx.x == 0) {
      const int32_t index = 0x7fffffff - static_cast<int32_t>(best & 0xffffffffu);
      top_tokens[r * top_k + j] = index;
      top_logprobs[r * top_k + j] = (to_float(row[index]) - m) - log_sum;
    }
  }
}

template <typename T>
void launch_logprobs(const void *logits, int64_t row_stride, int32_t rows, int32_t columns, const int64_t *tokens,
                     float *logprobs, float *entropy, float *top_logprobs, int64_t *top_tokens, int32_t top_k,
                     hipStream_t stream) {
  hipLaunchKernelGGL((token_logprobs_kernel<T>), dim3(static_cast<unsigned>(rows)), dim3(kThreads), 0, stream,
                     static_cast<const T *>(logits), row_stride, columns, tokens, logprobs, entropy, top_logprobs,
                     top_tokens, top_k);
}

}  // namespace
}  // namespace tf

extern "C" int32_t tf_token_logprobs(const void *logits, int64_t row_stride, int32_t rows, int32_t columns,
                                     const int64_t *tokens, float *logprobs, float *entropy, float *top_logprobs,
                                     int64_t *top_tokens, int32_t top_k, int32_t dtype, void *stream) {
  using namespace tf;
  clear_error();
  if (!valid_dtype(dtype)) return fail(TF_ERROR_INVALID_ARGUMENT, "unsupported dtype code");
  if (rows < 0) return fail(TF_ERROR_INVALID_ARGUMENT, "rows must be non-negative");
  if (columns < 1) return fail(TF_ERROR_INVALID_ARGUMENT, "log probabilities need at least one column");
  if (row_stride < columns) return fail(TF_ERROR_INVALID_ARGUMENT, "row stride is shorter than the rows");
  if (top_k < 0 || top_k > kMaxTop || top_k > columns)
    return fail(TF_ERROR_INVALID_ARGUMENT, "top_k must lie between 0 and 32 and not exceed the columns");
  if (rows == 0) return TF_SUCCESS;
  if (!logits || !tokens || !logprobs || !entropy || (top_k > 0 && (!top_logprobs || !top_tokens)))
    return fail(TF_ERROR_INVALID_ARGUMENT, "null tensor pointer");
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto launch = dtype == TF_DTYPE_FLOAT32   ? launch_logprobs<float>
                : dtype == TF_DTYPE_FLOAT16 ? launch_logprobs<_Float16>
                                            : launch_logprobs<__bf16>;
  launch(logits, row_stride, rows, columns, tokens, logprobs, entropy, top_logprobs, top_tokens, top_k, s);
  return check_launch("token_logprobs");
}
