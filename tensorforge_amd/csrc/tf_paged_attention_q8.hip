// Paged GQA decode attention over the 8-bit cache (tf_cache_q8.hip): one
// query token per row, keys and values as e4m3 codes with a power-of-two
// scale for each page and kv head.
//
// One workgroup per (row, kv head, partition); its wavefronts take 64 tokens,
// four tiles of 16, in turn, and every code goes from HBM to the registers it
// is multiplied in.  Scores S^T = K Q^T and outputs O^T = V^T P^T run on
// v_mfma_f32_16x16x32_bf16 with up to 16 query heads as the columns:
//
//  * V^T is stored as the operand wants it: lane (d, q) loads the 16 tokens of
//    tile q in dimension d.  So lane (head, q) has to hold the weights of tile
//    q's 16 tokens.
//  * The four score products of a block therefore take their 16 rows from all
//    four tiles: row 4 q + i of product r is token 4 r + i of tile q, and lane
//    (head, q) gets rows 4 q .. 4 q + 3.  No value crosses lanes between the
//    products but the maximum.
//
// e4m3 is exact in bf16 (v_cvt_scalef32_pk_bf16_fp8), a V code with its
// scale applied too; the K scale of a lane's tile multiplies its scores in
// fp32.  Queries and weights in bf16 parts: one for bf16 queries (p rounds to
// 2^-8, as in the 16-bit attention), two for fp16 (q exact, p 2^-16), three
// for fp32 (q and p 2^-24), the parts' products summed in fp32.
//
// Base-2 online softmax: a wavefront keeps the running maximum m of the scores
// (times log2 e), the sum l of exp2(s - m) and the unnormalised output; the
// wavefronts' meet in LDS.  Several partitions per row leave (m, l, numerator)
// for tf_paged_gqa_decode_merge.
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

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// Eight codes, in two words, times a power of two.
__device__ __forceinline__ bf16x8 decode8(uint32_t low, uint32_t high, float scale) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(low, scale, false);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(low, scale, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(high, scale, false);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(high, scale, true);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

template <typename T>
constexpr int kParts = sizeof(T) == 4 ? 3 : (__is_same(T, _Float16) ? 2 : 1);

// x as the sum of PARTS bf16 values (the last one rounded).
template <int PARTS>
__device__ __forceinline__ void split_parts(const float (&x)[8], bf16x8 (&parts)[PARTS]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    float rest = x[j];
#pragma unroll
    for (int i = 0; i < PARTS; ++i) {
      parts[i][j] = static_cast<__bf16>(rest);
      if (i + 1 < PARTS) rest -= static_cast<float>(parts[i][j]);
    }
  }
}

__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// Combine a value over the four lanes (head, 0..3); every lane gets the result.
template <typename F>
__device__ __forceinline__ float over_quads(float v, F combine) {
  uint32_t bits = __builtin_bit_cast(uint32_t, v);
  const auto halves = __builtin_amdgcn_permlane32_swap(bits, bits, false, false);
  const uint32_t low = halves[0], high = halves[1];
  v = combine(__builtin_bit_cast(float, low), __builtin_bit_cast(float, high));
  bits = __builtin_bit_cast(uint32_t, v);
  const auto rows = __builtin_amdgcn_permlane16_swap(bits, bits, false, false);
  const uint32_t even = rows[0], odd = rows[1];
  return combine(__builtin_bit_cast(float, even), __builtin_bit_cast(float, odd));
}

__device__ __forceinline__ float scale_of(uint32_t byte) { return __builtin_bit_cast(float, byte << 23); }

// What a wavefront loads of 64 tokens.
template <int DMAX>
struct Block {
  u32x4 k[4][DMAX / 64];
  u32x4 v[DMAX / 16];
  uint32_t k_scale, v_scale;
  int32_t tokens;  // of this lane's tile that count
};

// DMAX: head_dim, or with GUARD any head_dim up to it.
template <typename T, int DMAX, bool GUARD>
__global__ void __launch_bounds__(512) paged_decode_q8_kernel(Q8Params p) {
  constexpr int PARTS = kParts<T>;
  constexpr int KU = DMAX / 64;  // 16-byte loads of a key: 64 dimensions each
  constexpr int DT = DMAX / 16;  // tiles of the output
  constexpr bool AHEAD = DMAX <= 128;  // the next block is loaded before this one is used
  extern __shared__ float merged[];    // [wavefronts][heads][D + 4]
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int waves = blockDim.x >> 6;
  const int col = lane & 15;
  const int quad = lane >> 4;
  const int32_t D = GUARD ? p.head_dim : DMAX;
  const int32_t head_tiles = (p.group + 15) / 16;
  const int32_t h = blockIdx.x / head_tiles;
  const int32_t g0 = (blockIdx.x - h * head_tiles) * 16;
  const int32_t b = blockIdx.y;
  const int32_t split = blockIdx.z;
  const int32_t heads = min(16, p.group - g0);
  const int32_t qh0 = h * p.group + g0;

  int32_t ctx = p.context_lengths[b];
  ctx = ctx < 0 ? 0 : (ctx > p.max_tokens ? p.max_tokens : ctx);
  const int32_t begin = static_cast<int32_t>(min(static_cast<int64_t>(split) * p.split_size, static_cast<int64_t>(ctx)));
  const int32_t end = ctx - begin < p.split_size ? ctx : begin + p.split_size;
  if (begin >= end) {
    if (p.num_splits == 1) {
      T *out = static_cast<T *>(p.output) + (static_cast<int64_t>(b) * p.query_heads + qh0) * D;
      for (int i = threadIdx.x; i < heads * D; i += blockDim.x) out[i] = from_float<T>(0.f);
    }
    return;
  }

  // Queries: lane (head, quad) holds dimensions 64 u + 16 quad .. + 15.
  bf16x8 q[KU][2][PARTS];
  const T *query = static_cast<const T *>(p.query) + (static_cast<int64_t>(b) * p.query_heads + qh0 + min(col, heads - 1)) * D;
#pragma unroll
  for (int u = 0; u < KU; ++u)
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      float x[8];
      const int32_t d = 64 * u + 16 * quad + 8 * half;
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = !GUARD || d < D ? to_float(query[d + j]) : 0.f;
      split_parts<PARTS>(x, q[u][half]);
    }

  // A tile is 16 tokens of a page; `per_page` of them in a page.
  const int32_t per_page = p.block_size >> 4;
  const int32_t *table = p.block_tables + static_cast<int64_t>(b) * p.table_width;
  const int64_t page_bytes = static_cast<int64_t>(p.kv_heads) * p.block_size * D;
  const int64_t head_offset = static_cast<int64_t>(h) * p.block_size * D;
  struct Place {
    int32_t page, sub;  // page -1: none
  };
  auto place_of = [&](int32_t base) {
    Place at{-1, 0};
    const int32_t t = base + 16 * quad;
    if (base < end && t < end) {
      const int32_t tile = t >> 4;
      const int32_t logical = per_page == 1 ? tile : tile / per_page;
      at.page = table[logical];
      at.sub = per_page == 1 ? 0 : tile - logical * per_page;
    }
    return at;
  };
  auto load = [&](Block<DMAX> &blk, Place at, int32_t base) {
    if (base >= end) return;
    const bool inside = at.page >= 0 && at.page < p.num_blocks;
    blk.tokens = inside ? min(16, end - (base + 16 * quad)) : 0;
    const int32_t page = inside ? at.page : 0;  // loaded all the same, and masked
    const int32_t sub = inside ? at.sub : 0;
    const int64_t scale_at = static_cast<int64_t>(page) * p.kv_heads + h;
    blk.k_scale = p.key_scales[scale_at];
    blk.v_scale = p.value_scales[scale_at];
    const int from = lane & 12;  // lane (0, col / 4): the tile of this lane's key rows
    const int32_t k_page = __shfl(page, 4 * from, 64);
    const int32_t k_sub = __shfl(sub, 4 * from, 64);
    const uint8_t *key = p.key_cache + k_page * page_bytes + head_offset + (16 * k_sub + (col & 3)) * D + 16 * quad;
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int u = 0; u < KU; ++u) {
        if (!GUARD || 64 * u + 16 * quad < D)
          blk.k[r][u] = load_stream16<u32x4>(key + 4 * r * D + 64 * u);
        else
          blk.k[r][u] = u32x4{0, 0, 0, 0};
      }
    const uint8_t *value = p.value_cache + page * page_bytes + head_offset + col * p.block_size + 16 * sub;
#pragma unroll
    for (int j = 0; j < DT; ++j)
      if (!GUARD || 16 * j < D) blk.v[j] = load_stream16<u32x4>(value + 16 * j * p.block_size);
  };

  float m = kNegInf, l = 0.f;
  f32x4 acc[DT];
#pragma unroll
  for (int j = 0; j < DT; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};

  auto attend = [&](Block<DMAX> &blk, int32_t base) {
    if (base >= end) return;
    f32x4 s[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      s[r] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int u = 0; u < KU; ++u)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const bf16x8 a = decode8(blk.k[r][u][2 * half], blk.k[r][u][2 * half + 1], 1.f);
#pragma unroll
          for (int i = PARTS - 1; i >= 0; --i) s[r] = mfma(a, q[u][half][i], s[r]);
        }
    }
    const float unit = scale_of(blk.k_scale) * p.scale_log2;
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[r][i] *= unit;
    const bool whole = __all(blk.tokens >= 16);
    if (!whole) {
      // Tokens behind the end or outside the cache: scores of -inf, values of 0
      // (their codes may be anything, NaN too).
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[r][i] = 4 * r + i < blk.tokens ? s[r][i] : kNegInf;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const int left = blk.tokens - 4 * w;
        const uint32_t keep = left >= 4 ? ~0u : (left <= 0 ? 0u : (1u << (8 * left)) - 1);
#pragma unroll
        for (int j = 0; j < DT; ++j) blk.v[j][w] &= keep;
      }
      if (blk.tokens <= 0) blk.v_scale = 127;
    }
    float top = kNegInf;
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int i = 0; i < 4; ++i) top = fmaxf(top, s[r][i]);
    top = over_quads(top, [](float x, float y) { return fmaxf(x, y); });
    const float next = fmaxf(m, top);
    const float shift = next == kNegInf ? 0.f : next;  // no token yet
    if (__any(next > m)) {
      const float alpha = __builtin_amdgcn_exp2f(m - shift);
      l *= alpha;
#pragma unroll
      for (int j = 0; j < DT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[j][i] *= alpha;
      m = next;
    }
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      float w[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        w[j] = __builtin_amdgcn_exp2f(s[2 * half + j / 4][j % 4] - shift);
        l += w[j];
      }
      bf16x8 weights[PARTS];
      split_parts<PARTS>(w, weights);
      const float v_unit = scale_of(blk.v_scale);
#pragma unroll
      for (int j = 0; j < DT; ++j) {
        if (GUARD && 16 * j >= D) break;
        const bf16x8 a = decode8(blk.v[j][2 * half], blk.v[j][2 * half + 1], v_unit);
#pragma unroll
        for (int i = PARTS - 1; i >= 0; --i) acc[j] = mfma(a, weights[i], acc[j]);
      }
    }
  };

  const int32_t step = 64 * waves;
  int32_t base = begin + 64 * wave;
  if constexpr (AHEAD) {
    Block<DMAX> first, second;
    Place ahead = place_of(base);
    load(first, ahead, base);
    ahead = place_of(base + step);
    for (; base < end; base += 2 * step) {
      load(second, ahead, base + step);
      ahead = place_of(base + 2 * step);
      attend(first, base);
      load(first, ahead, base + 2 * step);
      ahead = place_of(base + 3 * step);
      attend(second, base + step);
    }
  } else {
    for (; base < end; base += step) {
      Block<DMAX> blk;
      load(blk, place_of(base), base);
      attend(blk, base);
    }
  }
  l = over_quads(l, [](float x, float y) { return x + y; });

  // The wavefronts' states: row (wave, head) holds D numerators, m and l.
  const int pitch = D + 4;
  if (col < heads) {
    float *state = merged + (wave * heads + col) * pitch;
#pragma unroll
    for (int j = 0; j < DT; ++j) {
      if (GUARD && 16 * j >= D) break;
      *reinterpret_cast<f32x4 *>(state + 16 * j + 4 * quad) = acc[j];
    }
    if (quad == 0) {
      state[D] = m;
      state[D + 1] = l;
    }
  }
  __syncthreads();
  for (int item = threadIdx.x; item < heads * D; item += blockDim.x) {
    const int head = item / D;
    const int d = item - head * D;
    const float *from = merged + head * pitch;
    float top = from[D];
    for (int w = 1; w < waves; ++w) top = fmaxf(top, from[w * heads * pitch + D]);
    const float shift = top == kNegInf ? 0.f : top;
    float sum = 0.f, num = 0.f;
    for (int w = 0; w < waves; ++w) {
      const float *one = from + w * heads * pitch;
      const float weight = __builtin_amdgcn_exp2f(one[D] - shift);
      sum += weight * one[D + 1];
      num += weight * one[d];
    }
    const int64_t row = static_cast<int64_t>(b) * p.query_heads + qh0 + head;
    if (p.num_splits == 1) {
      static_cast<T *>(p.output)[row * D + d] = from_float<T>(sum == 0.f ? 0.f : num / sum);
    } else {
      const int64_t slot = row * p.num_splits + split;
      p.partial_acc[slot * p.partial_stride + d] = num;
      if (d == 0) {
        p.partial_max[slot] = top;
        p.partial_sum[slot] = sum;
      }
    }
  }
}

template <typename T, int DMAX, bool GUARD>
void launch_attention(const Q8Params &p, int32_t batch, int waves, hipStream_t stream) {
  // As many wavefronts as leave their states within 64 KB of LDS: three at
  // least (16 heads of 256 dimensions).
  const int state = (p.group < 16 ? p.group : 16) * (p.head_dim + 4) * static_cast<int>(sizeof(float));
  const int fit = 64 * 1024 / state;
  if (waves > fit) waves = fit;
  hipLaunchKernelGGL((paged_decode_q8_kernel<T, DMAX, GUARD>),
                     dim3(p.kv_heads * ((p.group + 15) / 16), batch, p.num_splits), dim3(64 * waves), waves * state,
                     stream, p);
}

template <typename T>
void launch_dims(const Q8Params &p, int32_t batch, int waves, hipStream_t stream) {
  if (p.head_dim == 64) return launch_attention<T, 64, false>(p, batch, waves, stream);
  if (p.head_dim == 128) return launch_attention<T, 128, false>(p, batch, waves, stream);
  if (p.head_dim < 64) return launch_attention<T, 64, true>(p, batch, waves, stream);
  if (p.head_dim < 128) return launch_attention<T, 128, true>(p, batch, waves, stream);
  return launch_attention<T, 256, true>(p, batch, waves, stream);
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
  if (static_cast<int64_t>(table_width) * block_size > 1 << 30)
    return fail(TF_ERROR_UNSUPPORTED, "block tables of more than 2^30 tokens");
  if (batch > 65535 || num_splits > 65535)
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
  const int blocks = ((split_size < p.max_tokens ? split_size : p.max_tokens) + 63) / 64;
  const int waves = blocks < 1 ? 1 : (blocks < 8 ? blocks : 8);
  switch (dtype) {
    case TF_DTYPE_FLOAT32: launch_dims<float>(p, batch, waves, s); break;
    case TF_DTYPE_FLOAT16: launch_dims<_Float16>(p, batch, waves, s); break;
    default: launch_dims<__bf16>(p, batch, waves, s); break;
  }
  if (int32_t st = check_launch("paged_gqa_decode_q8")) return st;
  if (num_splits == 1) return TF_SUCCESS;
  return tf_paged_gqa_decode_merge(partial_max, partial_sum, partial_accumulator, context_lengths, output,
                                   partial_capacity, partial_row_stride, batch, query_heads, head_dim, split_size,
                                   num_splits, p.max_tokens, dtype, stream);
}
