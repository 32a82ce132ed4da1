// The 8-bit paged KV cache: append and read-back of token rows.
//
// Storage.  One page of one kv head is a contiguous tile of e4m3 codes, keys
// token-major [block_size][head_dim] and values dimension-major
// [head_dim][block_size], with one power-of-two scale each: value = code *
// 2^(byte - 127).  In this order a wavefront loads 16 tokens of a head as 16
// bytes per lane straight into the matrix operands of the attention products
// (K as rows of tokens, V as rows of dimensions), with no transpose between.
//
// Append.  Rows of one call that stand next to each other and fill a page in
// ascending order form a run (one token of a decode lane, or up to a page of
// a prompt).  For a run, t is the smallest integer >= -126 with
// max |finite x| <= 448 * 2^t.  A run that starts at offset 0 begins its page
// and sets the scale to 2^t; another raises the page's scale to 2^t where
// that is larger, and rounds the page's codes to it (exact but for codes that
// become subnormal).  Powers of two keep that requantisation, and every
// decode to bf16, free of rounding.
#include "tf_common.hpp"
#include "tf_q8.hpp"

namespace tf {
namespace {

struct Slots {
  const int32_t *physical_blocks;
  const int32_t *block_offsets;
  const int32_t *active_mask;  // null: every row
  int32_t rows;
  int32_t num_blocks;
  int32_t block_size;
  __device__ __forceinline__ bool valid(int32_t r, int32_t &block, int32_t &offset) const {
    block = physical_blocks[r];
    offset = block_offsets[r];
    return (!active_mask || active_mask[r] != 0) && block >= 0 && block < num_blocks && offset >= 0 &&
           offset < block_size;
  }
};

// Rows of the run that starts at row r, 0 when r is no start (its slot is not
// one, or it continues the row before).  Called by a whole wavefront.
__device__ __forceinline__ int32_t run_length(const Slots &s, int32_t r, int32_t &block, int32_t &offset) {
  if (!s.valid(r, block, offset)) return 0;
  int32_t other, at;
  if (r > 0 && s.valid(r - 1, other, at) && other == block && at + 1 == offset) return 0;
  const int lane = threadIdx.x & 63;
  int32_t n = 1;
  for (int32_t base = 1; base < s.block_size - offset; base += 64) {
    const int32_t next = base + lane;
    bool same = false;
    if (next < s.block_size - offset && next < s.rows - r)
      same = s.valid(r + next, other, at) && other == block && at == offset + next;
    const unsigned long long hits = __ballot(same);
    const int run = ~hits == 0 ? 64 : __builtin_ctzll(~hits);
    n += run;
    if (run < 64) break;
  }
  return n;
}

// One workgroup per (row, kv head): wavefront 0 stores the keys, wavefront 1
// the values, lanes across the head's dimensions.
template <typename T>
__global__ void __launch_bounds__(128)
kv_write_q8_kernel(const T *__restrict__ keys, const T *__restrict__ values, uint8_t *__restrict__ key_cache,
                   uint8_t *__restrict__ value_cache, uint8_t *__restrict__ key_scales,
                   uint8_t *__restrict__ value_scales, Slots slots, int32_t kv_heads, int32_t head_dim) {
  const int32_t r = blockIdx.x;
  const int32_t h = blockIdx.y;
  const int lane = threadIdx.x & 63;
  const bool is_value = threadIdx.x >= 64;
  int32_t block, offset;
  const int32_t n = run_length(slots, r, block, offset);
  if (n == 0) return;
  const T *src = (is_value ? values : keys) + (static_cast<int64_t>(r) * kv_heads + h) * head_dim;
  const int64_t row_stride = static_cast<int64_t>(kv_heads) * head_dim;
  const int64_t tile = static_cast<int64_t>(block) * kv_heads + h;
  uint8_t *scale = (is_value ? value_scales : key_scales) + tile;
  const int32_t page = slots.block_size;
  uint8_t *dst = (is_value ? value_cache : key_cache) + tile * page * head_dim;
  const int32_t dim_step = is_value ? page : 1;
  const int32_t token_step = is_value ? 1 : head_dim;

  uint32_t largest = 0;
  for (int32_t t = 0; t < n; ++t)
    for (int32_t d = lane; d < head_dim; d += 64) largest = max(largest, finite_bits(to_float(src[t * row_stride + d])));
  int32_t exponent = smallest_exponent(wave_umax(largest));
  if (offset > 0) {
    const int32_t old = static_cast<int32_t>(*scale) - 127;
    if (old < exponent) {
      for (int32_t i = lane; i < page * head_dim; i += 64)
        dst[i] = encode(ldexpf(decode(dst[i]), old - exponent));
      __threadfence_block();  // before other lanes store the new codes
    } else {
      exponent = old;
    }
  }
  if (lane == 0) *scale = static_cast<uint8_t>(exponent + 127);
  for (int32_t t = 0; t < n; ++t)
    for (int32_t d = lane; d < head_dim; d += 64)
      dst[d * dim_step + (offset + t) * token_step] = encode_scaled(to_float(src[t * row_stride + d]), exponent);
}

// One workgroup per (row, kv head), as in the append.
template <typename T>
__global__ void __launch_bounds__(128)
kv_read_q8_kernel(const uint8_t *__restrict__ key_cache, const uint8_t *__restrict__ value_cache,
                  const uint8_t *__restrict__ key_scales, const uint8_t *__restrict__ value_scales,
                  T *__restrict__ keys, T *__restrict__ values, Slots slots, int32_t kv_heads, int32_t head_dim) {
  const int32_t r = blockIdx.x;
  const int32_t h = blockIdx.y;
  const int lane = threadIdx.x & 63;
  const bool is_value = threadIdx.x >= 64;
  T *dst = (is_value ? values : keys) + (static_cast<int64_t>(r) * kv_heads + h) * head_dim;
  int32_t block, offset;
  if (!slots.valid(r, block, offset)) {
    for (int32_t d = lane; d < head_dim; d += 64) dst[d] = from_float<T>(0.f);
    return;
  }
  const int64_t tile = static_cast<int64_t>(block) * kv_heads + h;
  const int32_t page = slots.block_size;
  const uint8_t *src = (is_value ? value_cache : key_cache) + tile * page * head_dim;
  const int32_t exponent = static_cast<int32_t>((is_value ? value_scales : key_scales)[tile]) - 127;
  for (int32_t d = lane; d < head_dim; d += 64)
    dst[d] = from_float<T>(ldexpf(decode(is_value ? src[d * page + offset] : src[offset * head_dim + d]), exponent));
}

int32_t check_cache(const void *keys, const void *values, const void *key_cache, const void *value_cache,
                    const void *key_scales, const void *value_scales, const int32_t *physical_blocks,
                    const int32_t *block_offsets, int32_t rows, int32_t kv_heads, int32_t head_dim,
                    int32_t num_blocks, int32_t block_size, int32_t dtype) {
  if (!valid_dtype(dtype)) return fail(TF_ERROR_INVALID_ARGUMENT, "unsupported dtype code");
  if (int32_t s = check_q8_geometry(kv_heads, head_dim, num_blocks, block_size)) return s;
  if (rows < 0) return fail(TF_ERROR_INVALID_ARGUMENT, "rows must be non-negative");
  if (kv_heads > 65535) return fail(TF_ERROR_UNSUPPORTED, "grid too large");
  if (!key_cache || !value_cache || !key_scales || !value_scales)
    return fail(TF_ERROR_INVALID_ARGUMENT, "null tensor pointer");
  if (rows > 0 && (!keys || !values)) return fail(TF_ERROR_INVALID_ARGUMENT, "null tensor pointer");
  if (rows > 0 && (!physical_blocks || !block_offsets))
    return fail(TF_ERROR_INVALID_ARGUMENT, "null control vector");
  if ((reinterpret_cast<uintptr_t>(key_cache) | reinterpret_cast<uintptr_t>(value_cache)) % 16 != 0)
    return fail(TF_ERROR_INVALID_ARGUMENT, "cache tensors must be 16-byte aligned");
  return TF_SUCCESS;
}

template <typename T>
void launch_write(const void *keys, const void *values, void *key_cache, void *value_cache, void *key_scales,
                  void *value_scales, const Slots &slots, int32_t kv_heads, int32_t head_dim, hipStream_t s) {
  hipLaunchKernelGGL((kv_write_q8_kernel<T>), dim3(slots.rows, kv_heads), dim3(128), 0, s,
                     static_cast<const T *>(keys), static_cast<const T *>(values),
                     static_cast<uint8_t *>(key_cache), static_cast<uint8_t *>(value_cache),
                     static_cast<uint8_t *>(key_scales), static_cast<uint8_t *>(value_scales), slots, kv_heads,
                     head_dim);
}

template <typename T>
void launch_read(const void *key_cache, const void *value_cache, const void *key_scales, const void *value_scales,
                 void *keys, void *values, const Slots &slots, int32_t kv_heads, int32_t head_dim, hipStream_t s) {
  hipLaunchKernelGGL((kv_read_q8_kernel<T>), dim3(slots.rows, kv_heads), dim3(128), 0, s,
                     static_cast<const uint8_t *>(key_cache), static_cast<const uint8_t *>(value_cache),
                     static_cast<const uint8_t *>(key_scales), static_cast<const uint8_t *>(value_scales),
                     static_cast<T *>(keys), static_cast<T *>(values), slots, kv_heads, head_dim);
}

}  // namespace
}  // namespace tf

extern "C" int32_t tf_paged_kv_write_token_q8(
    const void *keys, const void *values, void *key_cache, void *value_cache, void *key_scales, void *value_scales,
    const int32_t *physical_blocks, const int32_t *block_offsets, const int32_t *active_mask, int32_t rows,
    int32_t kv_heads, int32_t head_dim, int32_t num_blocks, int32_t block_size, int32_t dtype, void *stream) {
  using namespace tf;
  clear_error();
  if (int32_t s = check_cache(keys, values, key_cache, value_cache, key_scales, value_scales, physical_blocks,
                              block_offsets, rows, kv_heads, head_dim, num_blocks, block_size, dtype))
    return s;
  if (rows == 0) return TF_SUCCESS;
  if (!active_mask) return fail(TF_ERROR_INVALID_ARGUMENT, "null control vector");
  const Slots slots{physical_blocks, block_offsets, active_mask, rows, num_blocks, block_size};
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto launch = dtype == TF_DTYPE_FLOAT32   ? launch_write<float>
                : dtype == TF_DTYPE_FLOAT16 ? launch_write<_Float16>
                                            : launch_write<__bf16>;
  launch(keys, values, key_cache, value_cache, key_scales, value_scales, slots, kv_heads, head_dim, s);
  return check_launch("paged_kv_write_token_q8");
}

extern "C" int32_t tf_paged_kv_read_token_q8(
    const void *key_cache, const void *value_cache, const void *key_scales, const void *value_scales,
    const int32_t *physical_blocks, const int32_t *block_offsets, void *keys, void *values, int32_t rows,
    int32_t kv_heads, int32_t head_dim, int32_t num_blocks, int32_t block_size, int32_t dtype, void *stream) {
  using namespace tf;
  clear_error();
  if (int32_t s = check_cache(keys, values, key_cache, value_cache, key_scales, value_scales, physical_blocks,
                              block_offsets, rows, kv_heads, head_dim, num_blocks, block_size, dtype))
    return s;
  if (rows == 0) return TF_SUCCESS;
  const Slots slots{physical_blocks, block_offsets, nullptr, rows, num_blocks, block_size};
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto launch = dtype == TF_DTYPE_FLOAT32   ? launch_read<float>
                : dtype == TF_DTYPE_FLOAT16 ? launch_read<_Float16>
                                            : launch_read<__bf16>;
  launch(key_cache, value_cache, key_scales, value_scales, keys, values, slots, kv_heads, head_dim, s);
  return check_launch("paged_kv_read_token_q8");
}
