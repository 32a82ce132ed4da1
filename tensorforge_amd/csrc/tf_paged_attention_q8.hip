// Paged GQA decode attention over the 8-bit cache (tf_cache_q8.hip): one
// query token per row, keys and values as e4m3 codes with a power-of-two
// scale for each page and kv head.
//
// Base-2 online softmax over the row's tokens, as in the 16-bit attention:
// a partition keeps the running maximum m of the scores (times log2 e), the
// sum l of exp2(s - m) and the unnormalised output.  Several partitions per
// row leave (m, l, numerator) for tf_paged_gqa_decode_merge.
#include "tf_common.hpp"
#include "tf_q8.hpp"

namespace tf {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNegInf = -__builtin_huge_valf();

struct Q8Params {
  const void *query;
  const uint8_t *key_cache;
  const uint8_t *value_cache;
  const uint8_t *key_scales;
  const uint8_t *value_scales;
  const int32_t *block_tables;
  const int32_t *context_lengths;
  void *output;
  float *partial_max;
  float *partial_sum;
  float *partial_acc;
  int32_t query_heads;
  int32_t kv_heads;
  int32_t group;
  int32_t head_dim;
  int32_t num_blocks;
  int32_t block_size;
  int32_t table_width;
  int32_t split_size;
  int32_t num_splits;
  int32_t partial_stride;
  int32_t max_tokens;  // min(num_splits * split_size, table_width * block_size)
  float scale_log2;
};

// One wavefront per (query head, row, partition): lanes across tokens for the
// scores, across dimensions for the output.
template <typename T>
__global__ void __launch_bounds__(64) paged_decode_q8_kernel(Q8Params p) {
  __shared__ float query[256];
  __shared__ float weights[64];
  __shared__ int32_t page_of[64];
  const int lane = threadIdx.x;
  const int32_t qh = blockIdx.x;
  const int32_t b = blockIdx.y;
  const int32_t split = blockIdx.z;
  const int32_t h = qh / p.group;
  const int32_t D = p.head_dim;
  const int64_t row = static_cast<int64_t>(b) * p.query_heads + qh;
  const T *q = static_cast<const T *>(p.query) + row * D;
  for (int d = lane; d < D; d += 64) query[d] = to_float(q[d]) * p.scale_log2;
  int32_t ctx = p.context_lengths[b];
  ctx = ctx < 0 ? 0 : (ctx > p.max_tokens ? p.max_tokens : ctx);
  const int32_t begin = split * p.split_size;
  const int32_t end = min(ctx, begin + p.split_size);
  __syncthreads();
  float m = kNegInf, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int32_t base = begin; base < end; base += 64) {
    const int32_t t = base + lane;
    int32_t page = -1;
    if (t < end) page = p.block_tables[static_cast<int64_t>(b) * p.table_width + t / p.block_size];
    if (page >= p.num_blocks) page = -1;
    const int32_t at = t % p.block_size;
    float s = kNegInf;
    if (page >= 0) {
      const int64_t tile = static_cast<int64_t>(page) * p.kv_heads + h;
      const uint8_t *k = p.key_cache + (tile * p.block_size + at) * D;
      s = 0.f;
      for (int d = 0; d < D; ++d) s += query[d] * decode(k[d]);
      s = ldexpf(s, static_cast<int32_t>(p.key_scales[tile]) - 127);
    }
    const float top = fmaxf(m, wave_max(s));
    const float shift = top == kNegInf ? 0.f : top;
    const float w = page >= 0 ? exp2f(s - shift) : 0.f;
    const float alpha = m == kNegInf ? 0.f : exp2f(m - shift);
    m = top;
    l = l * alpha + wave_sum(w);
    __syncthreads();
    weights[lane] = w;
    page_of[lane] = page;
    __syncthreads();
    for (int k = 0; k < 4; ++k) acc[k] *= alpha;
    for (int j = 0; j < 64; ++j) {
      if (page_of[j] < 0) continue;
      const int64_t tile = static_cast<int64_t>(page_of[j]) * p.kv_heads + h;
      const uint8_t *v = p.value_cache + tile * p.block_size * D + (base + j) % p.block_size;
      const float wj = ldexpf(weights[j], static_cast<int32_t>(p.value_scales[tile]) - 127);
      for (int k = 0; k < 4; ++k) {
        const int d = lane + 64 * k;
        if (d < D) acc[k] += wj * decode(v[static_cast<int64_t>(d) * p.block_size]);
      }
    }
  }
  if (p.num_splits == 1) {
    T *out = static_cast<T *>(p.output) + row * D;
    for (int k = 0; k < 4; ++k)
      if (lane + 64 * k < D) out[lane + 64 * k] = from_float<T>(l == 0.f ? 0.f : acc[k] / l);
    return;
  }
  if (begin >= ctx) return;
  const int64_t slot = row * p.num_splits + split;
  for (int k = 0; k < 4; ++k)
    if (lane + 64 * k < D) p.partial_acc[slot * p.partial_stride + lane + 64 * k] = acc[k];
  if (lane == 0) {
    p.partial_max[slot] = m;
    p.partial_sum[slot] = l;
  }
}

}  // namespace
}  // namespace tf

extern "C" int32_t tf_paged_gqa_decode_q8(
    const void *query, const void *key_cache, const void *value_cache, const void *key_scales,
    const void *value_scales, const int32_t *block_tables, const int32_t *context_lengths, void *output,
    float *partial_max, float *partial_sum, float *partial_accumulator, int64_t partial_capacity,
    int32_t partial_row_stride, int32_t batch, int32_t query_heads, int32_t kv_heads, int32_t head_dim,
    int32_t num_blocks, int32_t block_size, int32_t table_width, int32_t split_size, int32_t num_splits,
    float scale, int32_t dtype, void *stream) {
  using namespace tf;
  clear_error();
  if (!valid_dtype(dtype)) return fail(TF_ERROR_INVALID_ARGUMENT, "unsupported dtype code");
  if (int32_t s = check_q8_geometry(kv_heads, head_dim, num_blocks, block_size)) return s;
  if (batch < 0 || query_heads <= 0 || table_width <= 0)
    return fail(TF_ERROR_INVALID_ARGUMENT, "attention dimensions must be positive");
  if (query_heads % kv_heads != 0)
    return fail(TF_ERROR_INVALID_ARGUMENT, "query heads must be a multiple of kv heads");
  if (num_splits <= 0 || split_size <= 0 || split_size % 64 != 0)
    return fail(TF_ERROR_INVALID_ARGUMENT, "partitions must be a positive number of a multiple of 64 tokens");
  if (static_cast<int64_t>(table_width) * block_size > 0x7fffffff)
    return fail(TF_ERROR_UNSUPPORTED, "block tables of more than 2^31 - 1 tokens");
  if (batch > 65535 || num_splits > 65535 || query_heads > 65535)
    return fail(TF_ERROR_UNSUPPORTED, "grid too large");
  if (batch == 0) return TF_SUCCESS;
  if (!query || !key_cache || !value_cache || !key_scales || !value_scales || !block_tables || !context_lengths ||
      !output)
    return fail(TF_ERROR_INVALID_ARGUMENT, "null tensor pointer");
  if ((reinterpret_cast<uintptr_t>(key_cache) | reinterpret_cast<uintptr_t>(value_cache)) % 16 != 0)
    return fail(TF_ERROR_INVALID_ARGUMENT, "cache tensors must be 16-byte aligned");
  if (num_splits > 1) {
    if (!partial_max || !partial_sum || !partial_accumulator)
      return fail(TF_ERROR_INVALID_ARGUMENT, "several partitions need partial buffers");
    if (partial_capacity < static_cast<int64_t>(batch) * query_heads * num_splits || partial_row_stride < head_dim)
      return fail(TF_ERROR_INVALID_ARGUMENT, "partial buffers are too small");
  }
  const int64_t capacity = static_cast<int64_t>(table_width) * block_size;
  const int64_t reach = static_cast<int64_t>(num_splits) * split_size;
  const Q8Params p{query,
                   static_cast<const uint8_t *>(key_cache),
                   static_cast<const uint8_t *>(value_cache),
                   static_cast<const uint8_t *>(key_scales),
                   static_cast<const uint8_t *>(value_scales),
                   block_tables,
                   context_lengths,
                   output,
                   partial_max,
                   partial_sum,
                   partial_accumulator,
                   query_heads,
                   kv_heads,
                   query_heads / kv_heads,
                   head_dim,
                   num_blocks,
                   block_size,
                   table_width,
                   split_size,
                   num_splits,
                   partial_row_stride,
                   static_cast<int32_t>(reach < capacity ? reach : capacity),
                   scale * kLog2e};
  hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 grid(query_heads, batch, num_splits);
  switch (dtype) {
    case TF_DTYPE_FLOAT32: hipLaunchKernelGGL((paged_decode_q8_kernel<float>), grid, dim3(64), 0, s, p); break;
    case TF_DTYPE_FLOAT16: hipLaunchKernelGGL((paged_decode_q8_kernel<_Float16>), grid, dim3(64), 0, s, p); break;
    default: hipLaunchKernelGGL((paged_decode_q8_kernel<__bf16>), grid, dim3(64), 0, s, p); break;
  }
  if (int32_t st = check_launch("paged_gqa_decode_q8")) return st;
  if (num_splits == 1) return TF_SUCCESS;
  return tf_paged_gqa_decode_merge(partial_max, partial_sum, partial_accumulator, context_lengths, output,
                                   partial_capacity, partial_row_stride, batch, query_heads, head_dim, split_size,
                                   num_splits, p.max_tokens, dtype, stream);
}
