// Paged GQA decode attention over the 8-bit cache (tf_cache_q8.hip): one
// query token per row, keys and values as e4m3 codes with a power-of-two
// scale for each page and kv head.
//
// One workgroup per (row, kv head, partition); its wavefronts take 64 tokens,
// four tiles of 16, in turn, and every code reaches the lane that multiplies it
// in the order it is stored in.  Scores S^T = K Q^T and outputs O^T = V^T P^T run on
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
//
// Bound by HBM where rows are long: 4 rows of 8k to 32k tokens at 8 kv heads of
// 128 38 us with the merge, 5.0 TB/s; 72 rows of up to 2048 at 4 heads of 64
// 12.1-12.6 us, 2.9 TB/s, as the longest rows end last; one row of 300 5.6 us, of
// which 2.2 are an empty launch.
#include <algorithm>
#include <atomic>
#include <type_traits>

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

// One workgroup's part of a call: query heads [qh0, qh0 + heads) of row b, the
// tokens [begin, end) of a partition.
struct Part {
  int32_t b, h, qh0, heads, begin, end, split;
};

__device__ __forceinline__ Part part_of(const Q8Params &p) {
  Part w;
  const int32_t head_tiles = (p.group + 15) / 16;
  w.h = blockIdx.x / head_tiles;
  const int32_t g0 = (blockIdx.x - w.h * head_tiles) * 16;
  w.b = blockIdx.y;
  w.split = blockIdx.z;
  w.heads = min(16, p.group - g0);
  w.qh0 = w.h * p.group + g0;
  int32_t ctx = p.context_lengths[w.b];
  ctx = ctx < 0 ? 0 : (ctx > p.max_tokens ? p.max_tokens : ctx);
  w.begin = static_cast<int32_t>(min(static_cast<int64_t>(w.split) * p.split_size, static_cast<int64_t>(ctx)));
  w.end = ctx - w.begin < p.split_size ? ctx : w.begin + p.split_size;
  return w;
}

// A row without tokens is zeros; a partition without them leaves nothing.
template <typename T>
__device__ __forceinline__ void finish_empty(const Q8Params &p, const Part &w) {
  if (p.num_splits != 1) return;
  T *out = static_cast<T *>(p.output) + (static_cast<int64_t>(w.b) * p.query_heads + w.qh0) * p.head_dim;
  for (int i = threadIdx.x; i < w.heads * p.head_dim; i += blockDim.x) out[i] = from_float<T>(0.f);
}

// A wavefront's queries and running state.  DMAX: head_dim, or with GUARD any
// head_dim up to it.
template <typename T, int DMAX, bool GUARD>
struct Attention {
  static constexpr int PARTS = kParts<T>;
  static constexpr int KU = DMAX / 64;  // 16-byte pieces of a key per lane: 64 dimensions each
  static constexpr int DT = DMAX / 16;  // tiles of the output

  bf16x8 q[KU][2][PARTS];  // lane (head, quad): dimensions 64 u + 16 quad .. + 15
  float m = kNegInf, l = 0.f;
  f32x4 acc[DT];

  __device__ __forceinline__ void start(const Q8Params &p, const Part &w, int32_t D) {
    const int col = threadIdx.x & 15, quad = threadIdx.x >> 4 & 3;
    const T *query = static_cast<const T *>(p.query) +
                     (static_cast<int64_t>(w.b) * p.query_heads + w.qh0 + min(col, w.heads - 1)) * D;
#pragma unroll
    for (int u = 0; u < KU; ++u)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float x[8];
        const int32_t d = 64 * u + 16 * quad + 8 * half;
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = !GUARD || d < D ? to_float(query[d + j]) : 0.f;
        split_parts<PARTS>(x, q[u][half]);
        // In registers from here: left to their first use, the wait for them
        // would stand in the loop over blocks and hold its loads.
#pragma unroll
        for (int i = 0; i < PARTS; ++i) asm volatile("" : "+v"(q[u][half][i]));
      }
#pragma unroll
    for (int j = 0; j < DT; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  // 64 tokens: k[r] the key rows of product r, v[j] the values of dimensions
  // 16 j .. + 15; `tokens` of this lane's tile count, with the tile's scales.
  __device__ __forceinline__ void block(const u32x4 (&k)[4][KU], u32x4 (&v)[DT], uint32_t k_scale, uint32_t v_scale,
                                        int32_t tokens, float scale_log2, int32_t D) {
    f32x4 s[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      s[r] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int u = 0; u < KU; ++u)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const bf16x8 a = decode8(k[r][u][2 * half], k[r][u][2 * half + 1], 1.f);
#pragma unroll
          for (int i = PARTS - 1; i >= 0; --i) s[r] = mfma(a, q[u][half][i], s[r]);
        }
    }
    const float unit = scale_of(k_scale) * scale_log2;
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[r][i] *= unit;
    if (!__all(tokens >= 16)) {
      // Tokens behind the end or outside the cache: scores of -inf, values of 0
      // (their codes may be anything, NaN too).
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[r][i] = 4 * r + i < tokens ? s[r][i] : kNegInf;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const int left = tokens - 4 * w;
        const uint32_t keep = left >= 4 ? ~0u : (left <= 0 ? 0u : (1u << (8 * left)) - 1);
#pragma unroll
        for (int j = 0; j < DT; ++j) v[j][w] &= keep;
      }
      if (tokens <= 0) v_scale = 127;
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
    const float v_unit = scale_of(v_scale);
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
#pragma unroll
      for (int j = 0; j < DT; ++j) {
        if (!GUARD || 16 * j < D) {
          const bf16x8 a = decode8(v[j][2 * half], v[j][2 * half + 1], v_unit);
#pragma unroll
          for (int i = PARTS - 1; i >= 0; --i) acc[j] = mfma(a, weights[i], acc[j]);
        }
      }
    }
  }

  // The wavefronts' states meet in LDS (`merged`: [wavefronts][heads][D + 4], a
  // row the D numerators, l and m) and leave as output or partials.
  __device__ __forceinline__ void finish(const Q8Params &p, const Part &w, float *merged, int32_t D) {
    const int col = threadIdx.x & 15, quad = threadIdx.x >> 4 & 3;
    const int wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    l = over_quads(l, [](float x, float y) { return x + y; });
    const int pitch = D + 4;
    const int next = w.heads * pitch;
    float *state = merged + wave * next + col * pitch;
    float top = m;
    if (waves > 1) {  // every state to the largest maximum, so that the sums below are plain
      if (quad == 0 && col < w.heads) state[D + 1] = m;
      __syncthreads();
      for (int i = 0; i < waves; ++i) top = fmaxf(top, merged[i * next + min(col, w.heads - 1) * pitch + D + 1]);
      const float alpha = m == kNegInf ? 0.f : __builtin_amdgcn_exp2f(m - top);
      l *= l == 0.f ? 1.f : (m == kNegInf ? 1.f : alpha);
#pragma unroll
      for (int j = 0; j < DT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[j][i] *= alpha;
    }
    if (col < w.heads) {
#pragma unroll
      for (int j = 0; j < DT; ++j)
        if (!GUARD || 16 * j < D) *reinterpret_cast<f32x4 *>(state + 16 * j + 4 * quad) = acc[j];
      if (quad == 0) {
        state[D] = l;
        if (p.num_splits != 1 && wave == 0)
          p.partial_max[(static_cast<int64_t>(w.b) * p.query_heads + w.qh0 + col) * p.num_splits + w.split] = top;
      }
    }
    __syncthreads();
    const int quads = D / 4;
    for (int item = threadIdx.x; item < w.heads * quads; item += blockDim.x) {
      const int head = item / quads;
      const int d = 4 * (item - head * quads);
      const float *from = merged + head * pitch;
      float sum = 0.f;
      f32x4 num{0.f, 0.f, 0.f, 0.f};
      for (int i = 0; i < waves; ++i) {
        sum += from[i * next + D];
        num += *reinterpret_cast<const f32x4 *>(from + i * next + d);
      }
      const int64_t row = static_cast<int64_t>(w.b) * p.query_heads + w.qh0 + head;
      if (p.num_splits == 1) {
        T *out = static_cast<T *>(p.output) + row * D + d;
#pragma unroll
        for (int j = 0; j < 4; ++j) out[j] = from_float<T>(sum == 0.f ? 0.f : num[j] / sum);
      } else {
        const int64_t slot = row * p.num_splits + w.split;
#pragma unroll
        for (int j = 0; j < 4; ++j) p.partial_acc[slot * p.partial_stride + d + j] = num[j];
        if (d == 0) p.partial_sum[slot] = sum;
      }
    }
  }
};

// Any head_dim: the operands loaded straight to registers, block by block.
template <typename T, int DMAX>
__global__ void __launch_bounds__(512) paged_decode_q8_kernel(Q8Params p) {
  using A = Attention<T, DMAX, true>;
  extern __shared__ float merged[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15;
  const int quad = lane >> 4;
  const int32_t D = p.head_dim;
  const Part w = part_of(p);
  if (w.begin >= w.end) return finish_empty<T>(p, w);
  A state;
  state.start(p, w, D);
  // A tile is 16 tokens of a page.
  const int32_t per_page = p.block_size >> 4;
  const int32_t *table = p.block_tables + static_cast<int64_t>(w.b) * p.table_width;
  const int64_t page_bytes = static_cast<int64_t>(p.kv_heads) * p.block_size * D;
  const int64_t head_offset = static_cast<int64_t>(w.h) * p.block_size * D;
  for (int32_t base = w.begin + 64 * wave; base < w.end; base += blockDim.x) {
    const int32_t t = base + 16 * quad;
    int32_t page = -1, sub = 0, tokens = 0;
    if (t < w.end) {
      const int32_t tile = t >> 4;
      const int32_t logical = tile / per_page;
      page = table[logical];
      sub = tile - logical * per_page;
      tokens = min(16, w.end - t);
    }
    if (page < 0 || page >= p.num_blocks) page = sub = tokens = 0;  // page 0 is loaded and masked
    const int64_t scale_at = static_cast<int64_t>(page) * p.kv_heads + w.h;
    const uint32_t k_scale = p.key_scales[scale_at];
    const uint32_t v_scale = p.value_scales[scale_at];
    const int from = 4 * (lane & 12);  // lane (0, col / 4): the tile of this lane's key rows
    const int32_t k_page = __shfl(page, from, 64);
    const int32_t k_sub = __shfl(sub, from, 64);
    const uint8_t *key = p.key_cache + k_page * page_bytes + head_offset + (16 * k_sub + (col & 3)) * D + 16 * quad;
    u32x4 k[4][A::KU], v[A::DT];
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int u = 0; u < A::KU; ++u) {
        k[r][u] = u32x4{0, 0, 0, 0};
        if (64 * u + 16 * quad < D) k[r][u] = load_stream16<u32x4>(key + 4 * r * D + 64 * u);
      }
    const uint8_t *value = p.value_cache + page * page_bytes + head_offset + col * p.block_size + 16 * sub;
#pragma unroll
    for (int j = 0; j < A::DT; ++j) {
      v[j] = u32x4{0, 0, 0, 0};
      if (16 * j < D) v[j] = load_stream16<u32x4>(value + 16 * j * p.block_size);
    }
    state.block(k, v, k_scale, v_scale, tokens, p.scale_log2, D);
  }
  state.finish(p, w, merged, D);
}

// Tiles whose places and scales are in LDS together.
constexpr int kPanelTiles = 1024;

// A tile of 16 tokens: its page (-1: none), its place in the page, its scales.
struct Tile {
  int32_t page;
  uint16_t sub;
  uint8_t k_scale, v_scale;
};

// head_dim 64 and 128: whole tiles, 1 KB an instruction, by direct-to-LDS loads
// into a buffer of 64 tokens for each wavefront, refilled as soon as its
// operands are in registers.  Loaded in the operand layout, four rows from
// each of four tiles an instruction, the keys held the same kernel to
// 3.5 TB/s.  (Two and three buffers a wavefront: no case faster.)  The places
// of the partition's tiles are gathered first, their scales and the queries
// while the first blocks come in, so that the loop waits for nothing but its
// own blocks.
template <typename T, int D>
__global__ void __launch_bounds__(512) paged_decode_q8_stream_kernel(Q8Params p) {
  using A = Attention<T, D, false>;
  constexpr int kTileBytes = 16 * D;
  constexpr int kStage = 8 * kTileBytes;        // four tiles of keys, four of values
  constexpr int kPieces = D / 16;               // 16-byte pieces of a key
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int waves = blockDim.x >> 6;
  const int col = lane & 15;
  const int quad = lane >> 4;
  const int32_t per_page = p.block_size >> 4;
  const int32_t *table = p.block_tables + static_cast<int64_t>(blockIdx.y) * p.table_width;
  // The page of the partition's tile i, whatever the row's length: its load
  // does not wait for the length's.
  const int32_t first_tile = static_cast<int32_t>(
      min(static_cast<int64_t>(blockIdx.z) * p.split_size, static_cast<int64_t>(p.max_tokens)) >> 4);
  const int32_t last_tile = (p.max_tokens - 1) >> 4;
  auto page_of = [&](int32_t i) {
    const int32_t at = first_tile + i;
    if (at > last_tile) return -1;
    return table[per_page == 1 ? at : at / per_page];
  };
  const int32_t ahead = page_of(threadIdx.x);
  const Part w = part_of(p);
  if (w.begin >= w.end) return finish_empty<T>(p, w);
  unsigned char *ring = smem + wave * kStage;
  Tile *tiles = reinterpret_cast<Tile *>(smem + waves * kStage);
  const uint32_t lds0 = static_cast<uint32_t>(
      reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) unsigned char *)ring));
  const uint32_t page_bytes = static_cast<uint32_t>(p.kv_heads) * p.block_size * D;
  const uint32_t head_offset = static_cast<uint32_t>(w.h) * p.block_size * D;

  // Piece i of token t of tile q is kept at i ^ f(q, t), so that the 16 rows of
  // an operand read, four tokens of four tiles, lie in different banks.
  auto swizzle = [](int tile, int token) { return D == 64 ? tile : 2 * tile + (token >> 1 & 1); };
  uint32_t key_at[4][D / 64], value_at[D / 64];
#pragma unroll
  for (int half = 0; half < D / 64; ++half) {
    const int token = half * (1024 / D) + lane / kPieces;
#pragma unroll
    for (int i = 0; i < 4; ++i) key_at[i][half] = token * D + 16 * ((lane % kPieces) ^ swizzle(i, token));
    value_at[half] = (64 * half + lane) * p.block_size;
  }
  // A block's four tiles into the buffer.
  auto load = [&](const u32x4 (&four)[2]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int32_t page = __builtin_amdgcn_readfirstlane(static_cast<int32_t>(four[i / 2][2 * (i & 1)]));
      const uint32_t sub = __builtin_amdgcn_readfirstlane(four[i / 2][2 * (i & 1) + 1]) & 0xffffu;
      // (Scalar arithmetic: the bases below come from scalar instructions.)
      const uint64_t at = static_cast<uint64_t>(page < 0 ? 0u : static_cast<uint32_t>(page)) * page_bytes + head_offset;
      const uint8_t *key = p.key_cache + (at + sub * (16 * D));
      const uint8_t *value = p.value_cache + (at + 16 * sub);
#pragma unroll
      for (int half = 0; half < D / 64; ++half) {
        load_lds16<true>(key, key_at[i][half], __builtin_amdgcn_readfirstlane(lds0 + i * kTileBytes + half * 1024));
        load_lds16<true>(value, value_at[half],
                   __builtin_amdgcn_readfirstlane(lds0 + (4 + i) * kTileBytes + half * 1024));
      }
    }
  };
  auto tiles_of = [&](int32_t first, u32x4 (&four)[2]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) four[i] = *reinterpret_cast<const u32x4 *>(tiles + first + 2 * i);
  };

  A state;
  auto multiply = [&](int32_t first, int32_t tokens, int32_t next) {
    asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
    u32x4 k[4][A::KU], v[A::DT], four[2];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int tile = col >> 2, token = 4 * r + (col & 3);
#pragma unroll
      for (int u = 0; u < A::KU; ++u)
        k[r][u] = *reinterpret_cast<const u32x4 *>(ring + tile * kTileBytes + token * D +
                                                   16 * ((4 * u + quad) ^ swizzle(tile, token)));
    }
#pragma unroll
    for (int j = 0; j < A::DT; ++j)
      v[j] = *reinterpret_cast<const u32x4 *>(ring + (4 + quad) * kTileBytes + (16 * j + col) * 16);
    tiles_of(next >= 0 ? next : first, four);
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    const u32x2 mine = *reinterpret_cast<const u32x2 *>(tiles + first + quad);
    asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
    if (next >= 0) load(four);
    const int32_t page = static_cast<int32_t>(mine[0]);
    const uint32_t scales = mine[1] >> 16;
    const int32_t left = page >= 0 ? tokens - 16 * quad : 0;
    state.block(k, v, scales & 255u, scales >> 8, left < 16 ? left : 16, p.scale_log2, D);
  };

  for (int32_t panel = w.begin; panel < w.end; panel += 16 * kPanelTiles) {
    const int32_t tokens = min(w.end - panel, 16 * kPanelTiles);
    const int32_t blocks = (tokens + 63) >> 6;
    if (panel != w.begin) __syncthreads();  // the last panel's tiles are done with
    for (int32_t i = threadIdx.x; i < 4 * blocks; i += blockDim.x) {
      Tile tile{-1, 0, 127, 127};  // behind the end or outside: page 0 is loaded and masked
      if (16 * i < tokens) {
        const int32_t at = ((panel - w.begin) >> 4) + i;
        const int32_t page = at == static_cast<int32_t>(threadIdx.x) ? ahead : page_of(at);
        if (page >= 0 && page < p.num_blocks) {
          tile.page = page;
          tile.sub = static_cast<uint16_t>(per_page == 1 ? 0 : (first_tile + at) % per_page);
        }
      }
      tiles[i] = tile;
    }
    __syncthreads();
    const int32_t mine = (blocks - wave + waves - 1) / waves;
    auto first_of = [&](int32_t c) { return 4 * (wave + c * waves); };
    if (mine > 0) {
      u32x4 four[2];
      tiles_of(first_of(0), four);
      load(four);
    }
    for (int32_t i = threadIdx.x; i < 4 * blocks; i += blockDim.x) {
      const int32_t page = tiles[i].page;
      if (page < 0) continue;
      const int64_t scale_at = static_cast<int64_t>(page) * p.kv_heads + w.h;
      tiles[i].k_scale = p.key_scales[scale_at];
      tiles[i].v_scale = p.value_scales[scale_at];
    }
    if (panel == w.begin) state.start(p, w, D);
    __syncthreads();
    for (int32_t c = 0; c < mine; ++c)
      multiply(first_of(c), tokens - 16 * first_of(c), c + 1 < mine ? first_of(c + 1) : -1);
  }
  __syncthreads();  // every ring is done with
  state.finish(p, w, reinterpret_cast<float *>(smem), D);
}

// Bytes of LDS of one wavefront's state when the workgroup's meet.
int state_bytes(const Q8Params &p) {
  return (p.group < 16 ? p.group : 16) * (p.head_dim + 4) * static_cast<int>(sizeof(float));
}

dim3 attention_grid(const Q8Params &p, int32_t batch) {
  return dim3(p.kv_heads * ((p.group + 15) / 16), batch, p.num_splits);
}

template <typename T, int DMAX>
int32_t launch_any(const Q8Params &p, int32_t batch, int waves, hipStream_t stream) {
  // As many wavefronts as leave their states within 64 KB of LDS: three at
  // least (16 heads of 256 dimensions).
  const int fit = 64 * 1024 / state_bytes(p);
  if (waves > fit) waves = fit;
  hipLaunchKernelGGL((paged_decode_q8_kernel<T, DMAX>), attention_grid(p, batch), dim3(64 * waves),
                     waves * state_bytes(p), stream, p);
  return check_launch("paged_gqa_decode_q8");
}

template <typename T, int D>
int32_t launch_stream(const Q8Params &p, int32_t batch, int waves, hipStream_t stream) {
  auto kernel = paged_decode_q8_stream_kernel<T, D>;
  const int32_t tokens = p.split_size < p.max_tokens ? p.split_size : p.max_tokens;
  const int tiles = (tokens + 63) / 64 * 4 < kPanelTiles ? (tokens + 63) / 64 * 4 : kPanelTiles;
  const int ring = waves * 128 * D + tiles * static_cast<int>(sizeof(Tile));
  const int states = waves * state_bytes(p);
  const int lds = ring > states ? ring : states;
  if (lds > 64 * 1024) {
    // Raise the kernel's dynamic LDS limit once per device (a failure shows
    // up as a launch error).
    constexpr int kMaxDevices = 64;
    static std::atomic<bool> raised[kMaxDevices];
    int device = 0;
    if (hipGetDevice(&device) == hipSuccess && device >= 0 && device < kMaxDevices &&
        !raised[device].load(std::memory_order_acquire)) {
      if (hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                              160 * 1024) == hipSuccess)
        raised[device].store(true, std::memory_order_release);
    }
  }
  hipLaunchKernelGGL(kernel, attention_grid(p, batch), dim3(64 * waves), lds, stream, p);
  return check_launch("paged_gqa_decode_q8");
}

template <typename T>
int32_t launch_dims(const Q8Params &p, int32_t batch, int waves, hipStream_t stream) {
  if (p.head_dim == 64) return launch_stream<T, 64>(p, batch, waves, stream);
  if (p.head_dim == 128) return launch_stream<T, 128>(p, batch, waves, stream);
  if (p.head_dim < 64) return launch_any<T, 64>(p, batch, waves, stream);
  if (p.head_dim < 128) return launch_any<T, 128>(p, batch, waves, stream);
  return launch_any<T, 256>(p, batch, waves, stream);
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
  if (static_cast<int64_t>(kv_heads) * block_size * head_dim > 1 << 30)
    return fail(TF_ERROR_UNSUPPORTED, "pages of more than 2^30 codes");
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
  // Wavefronts of a workgroup: eight while every workgroup has a compute unit to
  // itself, four where units take several (64 rows of 1088 tokens, 4 kv heads of
  // 64, 256 workgroups: 10.6 us with eight, 11.1 with four; 72 rows to 2048,
  // 288: 15.4 and 13.9; sixteen were slower everywhere), none without a block.
  constexpr int64_t kUnits = 256;
  const int64_t groups = static_cast<int64_t>(kv_heads) * ((p.group + 15) / 16) * batch * num_splits;
  const int32_t blocks = ((split_size < p.max_tokens ? split_size : p.max_tokens) + 63) / 64;
  const int waves = std::min(groups <= kUnits ? 8 : 4, std::max(blocks, 1));
  const int32_t status = dtype == TF_DTYPE_FLOAT32   ? launch_dims<float>(p, batch, waves, s)
                         : dtype == TF_DTYPE_FLOAT16 ? launch_dims<_Float16>(p, batch, waves, s)
                                                     : launch_dims<__bf16>(p, batch, waves, s);
  if (status) return status;
  if (num_splits == 1) return TF_SUCCESS;
  return tf_paged_gqa_decode_merge(partial_max, partial_sum, partial_accumulator, context_lengths, output,
                                   partial_capacity, partial_row_stride, batch, query_heads, head_dim, split_size,
                                   num_splits, p.max_tokens, dtype, stream);
}
