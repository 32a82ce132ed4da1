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

// Whether row r has a slot, and whether it goes on the run of the row before.
__device__ __forceinline__ bool look(const Slots &s, int32_t r, int32_t &block, int32_t &offset, bool &goes_on) {
  goes_on = false;
  if (r < 0 || r >= s.rows || !s.valid(r, block, offset)) return false;
  int32_t other, at;
  goes_on = r > 0 && offset > 0 && s.valid(r - 1, other, at) && other == block && at + 1 == offset;
  return true;
}

// f(row, rows, block, offset) for every run that starts in rows [first, first +
// count), count <= 16.  Called by a whole wavefront: a lane looks at each of the
// next 64 rows, which hold every such run of pages up to 48 tokens.  Returns
// which of the rows have a slot.
template <typename F>
__device__ __forceinline__ uint32_t each_run(const Slots &s, int32_t first, int32_t count, F f) {
  const int lane = threadIdx.x & 63;
  int32_t block = 0, offset = 0;
  bool goes_on;
  const bool slot = look(s, first + lane, block, offset, goes_on);
  const unsigned long long more = __ballot(slot && goes_on);
  unsigned long long starts = __ballot(slot && !goes_on && lane < count);
  const unsigned long long has = __ballot(slot);
  while (starts) {
    const int at = __builtin_ctzll(starts);
    starts &= starts - 1;
    // (A run of 64 - at rows may go on behind them.)
    const unsigned long long rest = at == 63 ? 0 : more >> (at + 1);
    int32_t n = 1 + (~rest == 0 ? 63 : __builtin_ctzll(~rest));
    if (at + n >= 64) {
      bool on = true;
      while (on) {
        int32_t b, o;
        bool next;
        const bool is = look(s, first + at + n + lane, b, o, next);
        const unsigned long long hits = __ballot(is && next);
        const int run = ~hits == 0 ? 64 : __builtin_ctzll(~hits);
        n += run;
        on = run == 64;
      }
    }
    f(first + at, n, __builtin_amdgcn_readlane(block, at), __builtin_amdgcn_readlane(offset, at));
  }
  return static_cast<uint32_t>(has);
}

// 16 elements of a token from `at`, as 16-byte loads where the rows allow.
template <typename T>
__device__ __forceinline__ void load16(const T *at, bool whole, float (&x)[16]) {
  struct alignas(16) Vec {
    T v[16 / sizeof(T)];
  };
  constexpr int kPer = 16 / sizeof(T);
  if (whole) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)); ++i) {
      const Vec v = reinterpret_cast<const Vec *>(at)[i];
#pragma unroll
      for (int j = 0; j < kPer; ++j) x[kPer * i + j] = to_float(v.v[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j) x[j] = to_float(at[j]);
  }
}

template <typename T>
__device__ __forceinline__ void store16(T *at, bool whole, const float (&x)[16]) {
  struct alignas(16) Vec {
    T v[16 / sizeof(T)];
  };
  constexpr int kPer = 16 / sizeof(T);
  if (whole) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)); ++i) {
      Vec v;
#pragma unroll
      for (int j = 0; j < kPer; ++j) v.v[j] = from_float<T>(x[kPer * i + j]);
      reinterpret_cast<Vec *>(at)[i] = v;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j) at[j] = from_float<T>(x[j]);
  }
}

// A head's part of a page goes in groups of 16 tokens, from a multiple of 16,
// and a group in pieces of 16 dimensions of a token: piece q of a group's
// tokens is token q / (head_dim / 16) of them.  Lanes take pieces, PER at most.
struct Pieces {
  int32_t per_token, token, piece;
  __device__ __forceinline__ void at(int32_t q) {
    token = q / per_token;
    piece = q - token * per_token;
  }
};

// The transpose of a group's codes between pieces and whole dimensions, in a
// wavefront's own LDS [head_dim][16].
__device__ __forceinline__ void wave_order() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }

// One workgroup per (`count` rows, kv head): wavefront 0 stores the keys of the
// runs that start in them, wavefront 1 the values.  Per element (lanes across
// dimensions, two bytes in and one out) 8,058 rows at 4 heads of 64 took 14.6 us,
// by pieces 7.1 (12.4 MB, 2.2 of it an empty launch): latency of a run's scale,
// rows and stores, one run of a workgroup after the other.
template <typename T, int PER>
__global__ void __launch_bounds__(128)
kv_write_q8_kernel(const T *__restrict__ keys, const T *__restrict__ values, uint8_t *__restrict__ key_cache,
                   uint8_t *__restrict__ value_cache, uint8_t *__restrict__ key_scales,
                   uint8_t *__restrict__ value_scales, Slots slots, int32_t count, int32_t kv_heads,
                   int32_t head_dim, bool whole) {
  __shared__ __attribute__((aligned(16))) uint8_t turned[PER * 64 * 16];  // wavefront 1's
  const int32_t h = blockIdx.y;
  const int lane = threadIdx.x & 63;
  const bool is_value = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) != 0;
  const int64_t row_stride = static_cast<int64_t>(kv_heads) * head_dim;
  const int32_t page = slots.block_size;
  Pieces pieces{head_dim / 16, 0, 0};
  each_run(slots, blockIdx.x * count, count, [&](int32_t r, int32_t n, int32_t block, int32_t offset) {
    const T *src = (is_value ? values : keys) + r * row_stride + static_cast<int64_t>(h) * head_dim;
    const int64_t tile = static_cast<int64_t>(block) * kv_heads + h;
    uint8_t *scale = (is_value ? value_scales : key_scales) + tile;
    uint8_t *dst = (is_value ? value_cache : key_cache) + tile * page * head_dim;
    const int32_t end = offset + n;
    float x[PER][16];
    // Pieces of the group's tokens [low, high).
    auto load = [&](int32_t low, int32_t high) {
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int32_t q = lane + 64 * i;
        pieces.at(q);
        if (low + pieces.token < high) {
          load16(src + (low + pieces.token - offset) * row_stride + 16 * pieces.piece, whole, x[i]);
        } else {
#pragma unroll
          for (int j = 0; j < 16; ++j) x[i][j] = 0.f;
        }
      }
    };
    const int32_t old = offset > 0 ? static_cast<int32_t>(*scale) - 127 : kLowestExponent;
    const int32_t begin = offset & ~15;
    uint32_t largest = 0;
    for (int32_t g = begin; g < end; g += 16) {
      load(max(g, offset), min(g + 16, end));
#pragma unroll
      for (int i = 0; i < PER; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) largest = max(largest, finite_bits(x[i][j]));
    }
    const int32_t needed = smallest_exponent(wave_umax(largest));
    const int32_t exponent = max(old, needed);
    if (offset > 0 && old < needed) {
      for (int32_t i = lane; i < page * head_dim / 16; i += 64) {
        uint4 codes = reinterpret_cast<uint4 *>(dst)[i];
        uint32_t *words = reinterpret_cast<uint32_t *>(&codes);
#pragma unroll
        for (int w = 0; w < 4; ++w) words[w] = rescale4(words[w], old - exponent);
        reinterpret_cast<uint4 *>(dst)[i] = codes;
      }
      __threadfence_block();  // before other lanes store the new codes
    }
    if (lane == 0) *scale = static_cast<uint8_t>(exponent + 127);
    const bool again = end - begin > 16;
    for (int32_t g = begin; g < end; g += 16) {
      const int32_t low = max(g, offset), high = min(g + 16, end);
      if (again) load(low, high);
      if (is_value) wave_order();  // the last group's codes have been read
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int32_t q = lane + 64 * i;
        pieces.at(q);
        const int32_t token = low + pieces.token;
        if (token >= high) continue;
        uint4 codes;
        uint32_t *words = reinterpret_cast<uint32_t *>(&codes);
#pragma unroll
        for (int w = 0; w < 4; ++w)
          words[w] = encode4(x[i][4 * w], x[i][4 * w + 1], x[i][4 * w + 2], x[i][4 * w + 3], exponent);
        if (!is_value) {
          *reinterpret_cast<uint4 *>(dst + token * head_dim + 16 * pieces.piece) = codes;
        } else {
#pragma unroll
          for (int j = 0; j < 16; ++j)
            turned[(16 * pieces.piece + j) * 16 + token - g] = static_cast<uint8_t>(words[j / 4] >> (8 * (j % 4)));
        }
      }
      if (!is_value) continue;
      wave_order();
      for (int32_t d = lane; d < head_dim; d += 64) {
        if (high - low == 16) {
          *reinterpret_cast<uint4 *>(dst + static_cast<int64_t>(d) * page + g) =
              *reinterpret_cast<const uint4 *>(turned + 16 * d);
        } else {
          for (int32_t token = low; token < high; ++token) dst[d * page + token] = turned[16 * d + token - g];
        }
      }
    }
  });
}

// The same split over workgroups; rows without a slot become zeros.  8,058 rows
// at 4 heads of 64 to bf16 11.3 us (12.4 MB).
template <typename T, int PER>
__global__ void __launch_bounds__(128)
kv_read_q8_kernel(const uint8_t *__restrict__ key_cache, const uint8_t *__restrict__ value_cache,
                  const uint8_t *__restrict__ key_scales, const uint8_t *__restrict__ value_scales,
                  T *__restrict__ keys, T *__restrict__ values, Slots slots, int32_t count, int32_t kv_heads,
                  int32_t head_dim, bool whole) {
  __shared__ __attribute__((aligned(16))) uint8_t turned[16 * (PER * 64 + 16)];  // [16 tokens][head_dim + 16]
  const int32_t h = blockIdx.y;
  const int lane = threadIdx.x & 63;
  const bool is_value = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) != 0;
  const int64_t row_stride = static_cast<int64_t>(kv_heads) * head_dim;
  const int32_t page = slots.block_size;
  const int32_t pitch = head_dim + 16;
  T *out = (is_value ? values : keys) + static_cast<int64_t>(h) * head_dim;
  Pieces pieces{head_dim / 16, 0, 0};
  const int32_t first = blockIdx.x * count;
  const uint32_t has = each_run(slots, first, count, [&](int32_t r, int32_t n, int32_t block, int32_t offset) {
    const int64_t tile = static_cast<int64_t>(block) * kv_heads + h;
    const uint8_t *src = (is_value ? value_cache : key_cache) + tile * page * head_dim;
    const int32_t exponent = static_cast<int32_t>((is_value ? value_scales : key_scales)[tile]) - 127;
    const int32_t end = offset + n;
    for (int32_t g = offset & ~15; g < end; g += 16) {
      const int32_t low = max(g, offset), high = min(g + 16, end);
      if (is_value) {
        wave_order();  // the last group's codes have been read
        for (int32_t d = lane; d < head_dim; d += 64) {
          const uint4 codes = *reinterpret_cast<const uint4 *>(src + static_cast<int64_t>(d) * page + g);
          const uint32_t *words = reinterpret_cast<const uint32_t *>(&codes);
#pragma unroll
          for (int t = 0; t < 16; ++t) turned[t * pitch + d] = static_cast<uint8_t>(words[t / 4] >> (8 * (t % 4)));
        }
        wave_order();
      }
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int32_t q = lane + 64 * i;
        pieces.at(q);
        const int32_t token = low + pieces.token;
        if (token >= high) continue;
        const uint8_t *at = is_value ? turned + (token - g) * pitch : src + token * head_dim;
        const uint4 codes = *reinterpret_cast<const uint4 *>(at + 16 * pieces.piece);
        const uint32_t *words = reinterpret_cast<const uint32_t *>(&codes);
        float x[16];
#pragma unroll
        for (int w = 0; w < 4; ++w) decode4(words[w], exponent, x + 4 * w);
        store16(out + (r + token - offset) * row_stride + 16 * pieces.piece, whole, x);
      }
    }
  });
  uint32_t without = ~has & ((1u << min(count, slots.rows - first)) - 1);
  while (without) {
    const int64_t r = first + __builtin_ctz(without);
    without &= without - 1;
    for (int32_t d = lane; d < head_dim; d += 64) out[r * row_stride + d] = from_float<T>(0.f);
  }
}

// Rows of a workgroup.  A few rows are a decode step's lanes, each a run of its
// own that waits for its page: a workgroup each.  Many are prompts, whose runs
// are pages and start in every 16th row or less.  On MI355X, graph-timed, with
// 1 / 4 / 16 rows to a workgroup, 4 kv heads of 64 in pages of 16: write of 72
// rows 4.3 / 9.0 / 28 us, of 900 (chunks of prompts) 7.9 / 5.9 / 7.0, of 8,058
// 15.5 / 8.9 / 7.1; read of 595 rows 4.6 / 4.3 / 4.7, of 1,724 12.6 / 10.4 / 9.0,
// of 8,058 18.0 / 14.0 / 11.3.
inline int32_t rows_per_group(int32_t rows) { return rows <= 512 ? 1 : rows <= 1024 ? 4 : 16; }

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
  auto kernel = head_dim <= 64    ? kv_write_q8_kernel<T, 1>
                : head_dim <= 128 ? kv_write_q8_kernel<T, 2>
                                  : kv_write_q8_kernel<T, 4>;
  const int32_t count = rows_per_group(slots.rows);
  const bool whole = (reinterpret_cast<uintptr_t>(keys) | reinterpret_cast<uintptr_t>(values)) % 16 == 0;
  hipLaunchKernelGGL(kernel, dim3((slots.rows + count - 1) / count, kv_heads), dim3(128), 0, s,
                     static_cast<const T *>(keys), static_cast<const T *>(values),
                     static_cast<uint8_t *>(key_cache), static_cast<uint8_t *>(value_cache),
                     static_cast<uint8_t *>(key_scales), static_cast<uint8_t *>(value_scales), slots, count, kv_heads,
                     head_dim, whole);
}

template <typename T>
void launch_read(const void *key_cache, const void *value_cache, const void *key_scales, const void *value_scales,
                 void *keys, void *values, const Slots &slots, int32_t kv_heads, int32_t head_dim, hipStream_t s) {
  auto kernel = head_dim <= 64    ? kv_read_q8_kernel<T, 1>
                : head_dim <= 128 ? kv_read_q8_kernel<T, 2>
                                  : kv_read_q8_kernel<T, 4>;
  const int32_t count = rows_per_group(slots.rows);
  const bool whole = (reinterpret_cast<uintptr_t>(keys) | reinterpret_cast<uintptr_t>(values)) % 16 == 0;
  hipLaunchKernelGGL(kernel, dim3((slots.rows + count - 1) / count, kv_heads), dim3(128), 0, s,
                     static_cast<const uint8_t *>(key_cache), static_cast<const uint8_t *>(value_cache),
                     static_cast<const uint8_t *>(key_scales), static_cast<const uint8_t *>(value_scales),
                     static_cast<T *>(keys), static_cast<T *>(values), slots, count, kv_heads, head_dim, whole);
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
