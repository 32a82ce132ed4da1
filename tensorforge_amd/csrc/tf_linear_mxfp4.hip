// Decode projections by 4-bit weights: y = x . W^T for at most 64 rows, W in
// e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives) with a power-of-two
// scale (e8m0) for each 32 columns of K.
//   y[r][n] = sum_k x[r][k] * e2m1(code[n][k]) * 2^(scale[n][k / 32] - 127)
// in fp32, rounded once; with a residual, round(round(sum) + residual).
//
// The products run on v_mfma_f32_16x16x32 with 16 weight rows as the A operand
// and 16 rows of x as the B operand.  A lane's 16 bytes of a weight row are one
// group of 32 columns, so it has one scale; which columns meet in one
// instruction does not matter as long as x takes the same order: step s
// multiplies columns 8 s .. 8 s + 7 of each lane's group.
// v_cvt_scalef32_pk_bf16_fp4 turns two codes into bf16 with the scale applied,
// exactly, so nothing is left to do to the sums.
//
// Operands go through LDS.  Loaded in the operand layout (16 rows of 64 bytes
// an instruction, a scale byte from each) the same products were bound by the
// 53 B/ns at which a compute unit takes lines: 8 rows by 28672 x 4096 24 us,
// 64 by 2048 x 2048 11 us; through LDS 15.7 and 5.2.  At few rows HBM bounds
// (8 by 28672 x 4096 reads 4.0 TB/s), at many that rate still: x for every tile.
#include <atomic>
#include <type_traits>

#include "tf_common.hpp"

namespace tf {
namespace {

constexpr int32_t kMaxRows = 64;
constexpr int32_t kChunk = 256;  // columns of K a wavefront takes at a time: 128 bytes of a weight row
constexpr int32_t kPanel = 8192;  // columns of K whose scales are in LDS together
constexpr int32_t kXcds = 8;

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
  int32_t column_tiles, row_blocks;
  int32_t stream;        // weights by nontemporal loads
  int32_t scale_words;   // scale rows may be read as 32-bit words
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

// Chunks in flight per wavefront: what lets two workgroups of four share a
// compute unit's LDS.
constexpr int ring_stages(int stage_bytes) {
  const int fit = 60 * 1024 / (4 * stage_bytes);
  return fit < 1 ? 1 : (fit > 3 ? 3 : fit);
}

// Bytes from one row of a panel's scales to the next in LDS: an odd number of
// words, so that the rows of a read start in different banks.
__host__ __device__ constexpr int scale_pitch(int32_t k) {
  const int bytes = (k < kPanel ? k : kPanel) / 32;
  return 4 * ((bytes + 3) / 4 | 1);
}

// The scales of the tile's rows and of the columns [panel, end) to LDS.
template <int NT>
__device__ __forceinline__ void load_scales(const LinearParams &p, int32_t n0, int32_t panel, int32_t end,
                                            unsigned char *scales, int scale_row) {
  const int32_t bytes = (end - panel) / 32;
  if (p.scale_words) {
    const int32_t words = bytes / 4;
    for (int32_t i = threadIdx.x; i < 16 * NT * words; i += blockDim.x) {
      const int32_t row = i / words;
      const int64_t from = min(n0 + row, p.n - 1) * p.scale_stride + panel / 32;
      *reinterpret_cast<uint32_t *>(scales + row * scale_row + 4 * (i - row * words)) =
          *reinterpret_cast<const uint32_t *>(p.scales + from + 4 * (i - row * words));
    }
  } else {
    for (int32_t i = threadIdx.x; i < 16 * NT * bytes; i += blockDim.x) {
      const int32_t row = i / bytes;
      scales[row * scale_row + i - row * bytes] =
          p.scales[min(n0 + row, p.n - 1) * p.scale_stride + panel / 32 + i - row * bytes];
    }
  }
}

// The wavefronts' sums [waves][MR][NT][64] added in their order, rounded and stored.
template <typename T, int MR, int NT>
__device__ __forceinline__ void join(const LinearParams &p, const f32x4 *sums, int waves, int32_t m0, int32_t n0) {
  for (int item = threadIdx.x; item < MR * NT * 64; item += blockDim.x) {
    f32x4 sum = sums[item];
    for (int w = 1; w < waves; ++w) sum += sums[w * MR * NT * 64 + item];
    const int32_t tile = item >> 6;
    const int32_t r = m0 + 16 * (tile / NT) + (item & 15);
    const int32_t first = n0 + 16 * (tile % NT) + 4 * ((item >> 4) & 3);
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

// A workgroup computes a tile of 16 NT columns of y for 16 rows of x (XR of
// which are loaded), over all of K.  Its wavefronts take the chunks of K in
// turn, each through a ring of its own in LDS that direct-to-LDS loads fill,
// and their tiles meet in LDS in the wavefronts' order.  The tile's scales are
// read once, a panel of K at a time.
template <typename T, int XR, int NT>
__global__ void __launch_bounds__(512) linear_mxfp4_kernel(LinearParams p) {
  typedef typename Operand<T>::V V;
  constexpr int kWeightLoads = 2 * NT;  // 8 rows of 128 bytes each
  constexpr int kRowLoads = XR / 2;     // 2 rows of 512 bytes each
  constexpr int kLoads = kWeightLoads + kRowLoads;
  constexpr int kStage = 1024 * kLoads;
  constexpr int STAGES = ring_stages(kStage);
  const int scale_row = scale_pitch(p.k);
  static_assert(kLoads * STAGES <= 63, "vmcnt range");
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int waves = blockDim.x >> 6;
  const int col = lane & 15;
  const int quad = lane >> 4;
  // The row blocks of a column tile are workgroups of one die (id % 8), whose
  // L2 then holds its weights.
  const int32_t group = static_cast<int32_t>(blockIdx.x) / (kXcds * p.row_blocks);
  const int32_t in = static_cast<int32_t>(blockIdx.x) - group * kXcds * p.row_blocks;
  const int32_t tile = group * kXcds + in % kXcds;
  if (tile >= p.column_tiles) return;
  const int32_t n0 = tile * 16 * NT;
  const int32_t m0 = in / kXcds * 16;
  unsigned char *ring = smem + wave * (STAGES * kStage);
  unsigned char *scales = smem + waves * (STAGES * kStage);
  const uint32_t lds0 = static_cast<uint32_t>(
      reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) unsigned char *)ring));

  // 16-byte piece i of row r is kept at i ^ r (of 8 or 16 neighbours), so that
  // the rows of an operand read lie in different banks.
  const uint8_t *weight[kWeightLoads];
  const int weight_piece = (lane & 7) ^ (lane >> 3);
#pragma unroll
  for (int i = 0; i < kWeightLoads; ++i)
    weight[i] = p.weight + static_cast<int64_t>(min(n0 + 8 * i + (lane >> 3), p.n - 1)) * p.weight_stride;
  const T *x[kRowLoads];
  int row_piece[kRowLoads];
#pragma unroll
  for (int i = 0; i < kRowLoads; ++i) {
    const int row = 2 * i + (lane >> 5);
    x[i] = static_cast<const T *>(p.x) + static_cast<int64_t>(min(m0 + row, p.m - 1)) * p.x_stride;
    row_piece[i] = (lane & 31) ^ row;
  }
  auto load = [&](int32_t base, int stage) {
    // Pieces behind K read the row's last one and are not multiplied.
    const int32_t code = min(base / 2 + 16 * weight_piece, p.k / 2 - 16);
#pragma unroll
    for (int i = 0; i < kWeightLoads; ++i) {
      const uint32_t at = __builtin_amdgcn_readfirstlane(lds0 + stage * kStage + i * 1024);
      if (p.stream)
        load_lds16<true>(weight[i] + code, at);
      else
        load_lds16(weight[i] + code, at);
    }
#pragma unroll
    for (int i = 0; i < kRowLoads; ++i)
      load_lds16(x[i] + min(base + 8 * row_piece[i], p.k - 8),
                 __builtin_amdgcn_readfirstlane(lds0 + stage * kStage + (kWeightLoads + i) * 1024));
  };

  f32x4 acc[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};

  // One chunk, FLIGHT chunks being loaded behind it; NEXT >= 0: its buffer then
  // takes the chunk at NEXT (all operands are in registers before).
  auto multiply = [&](auto flight, int32_t base, int32_t panel, int stage, int32_t next) {
    asm volatile("s_waitcnt vmcnt(%0)" : : "n"(kLoads * decltype(flight)::value) : "memory");
    const unsigned char *at = ring + stage * kStage;
    u32x4 codes[2][NT];
    V rows[2][4];
    uint32_t exponent[2][NT];
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const int piece = 4 * g + quad;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        codes[g][t] = *reinterpret_cast<const u32x4 *>(at + (16 * t + col) * 128 + 16 * (piece ^ (col & 7)));
        exponent[g][t] = scales[(16 * t + col) * scale_row + (base - panel) / 32 + piece];
      }
      const int row = col & (XR - 1);
#pragma unroll
      for (int s = 0; s < 4; ++s)
        rows[g][s] = *reinterpret_cast<const V *>(at + kWeightLoads * 1024 + row * 512 + 16 * ((4 * piece + s) ^ row));
    }
    asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
    if (next >= 0) load(next, stage);
    if (base + kChunk > p.k) {  // groups behind K: zero on both sides, whatever x holds there
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        if (base + 32 * (4 * g + quad) < p.k) continue;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          codes[g][t] = u32x4{0, 0, 0, 0};
          exponent[g][t] = 127;
        }
#pragma unroll
        for (int s = 0; s < 4; ++s) rows[g][s] = V{0, 0, 0, 0, 0, 0, 0, 0};
      }
    }
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      if constexpr (__is_same(T, _Float16)) {
        // 0.5 * 2^-13 is fp16's smallest normal value, 6 * 2^13 below its
        // largest: outside, the weights take bf16's range and x two parts.
        bool wide = false;
#pragma unroll
        for (int t = 0; t < NT; ++t) wide |= exponent[g][t] - (127 - 13) > 26;
        if (__any(wide)) {
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            bf16x8 high, low;
            split(rows[g][s], high, low);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              const bf16x8 a =
                  Operand<__bf16>::decode(codes[g][t][s], __builtin_bit_cast(float, exponent[g][t] << 23));
              acc[t] = Operand<__bf16>::mfma(a, high, acc[t]);
              acc[t] = Operand<__bf16>::mfma(a, low, acc[t]);
            }
          }
          continue;
        }
      }
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int t = 0; t < NT; ++t)
          acc[t] = Operand<T>::mfma(
              Operand<T>::decode(codes[g][t][s], __builtin_bit_cast(float, exponent[g][t] << 23)), rows[g][s], acc[t]);
    }
  };

  for (int32_t panel = 0; panel < p.k; panel += kPanel) {
    const int32_t end = min(panel + kPanel, p.k);
    const int32_t chunks = (end - panel + kChunk - 1) / kChunk;
    const int32_t mine = (chunks - wave + waves - 1) / waves;
    auto base_of = [&](int32_t c) { return panel + (wave + c * waves) * kChunk; };
#pragma unroll
    for (int i = 0; i < STAGES; ++i)
      if (i < mine) load(base_of(i), i);
    load_scales<NT>(p, n0, panel, end, scales, scale_row);
    __syncthreads();
    int32_t c = 0;
    int stage = 0;
    auto step = [&](auto flight, bool more) {
      multiply(flight, base_of(c), panel, stage, more ? base_of(c + STAGES) : -1);
      stage = stage + 1 == STAGES ? 0 : stage + 1;
      ++c;
    };
    while (c + STAGES < mine) step(std::integral_constant<int, STAGES - 1>{}, true);
    if constexpr (STAGES >= 3)
      if (mine - c >= 3) step(std::integral_constant<int, 2>{}, false);
    if constexpr (STAGES >= 2)
      if (mine - c >= 2) step(std::integral_constant<int, 1>{}, false);
    if (mine - c >= 1) step(std::integral_constant<int, 0>{}, false);
    __syncthreads();  // the panel's scales and every ring are done with
  }

  f32x4 *sums = reinterpret_cast<f32x4 *>(smem);  // [wavefronts][NT][64]
#pragma unroll
  for (int t = 0; t < NT; ++t) sums[(wave * NT + t) * 64 + lane] = acc[t];
  __syncthreads();
  join<T, 1, NT>(p, sums, waves, m0, n0);
}

// The same products for 17 to 64 rows and many columns: a workgroup computes all
// 16 MR rows by 16 NT columns, so x is read once per 16 NT columns and not once
// per row block and tile.  The eight wavefronts fill one ring together, each
// takes an eighth of every chunk's columns for the whole tile, and a barrier a
// chunk says that the chunk is there and that the buffer of the one before is
// free.  A weight is decoded once for all rows.
template <typename T, int MR, int NT, int STAGES>
__global__ void __launch_bounds__(512) linear_mxfp4_rows_kernel(LinearParams p) {
  typedef typename Operand<T>::V V;
  constexpr int kWeightBytes = 2048 * NT;
  constexpr int kStage = kWeightBytes + 8192 * MR;
  constexpr int WAVES = 8;
  constexpr int kWeightLoads = 2 * NT;  // of 1024 bytes: 8 rows of 128 bytes
  constexpr int kMine = kWeightLoads / WAVES;
  constexpr int kExtra = kWeightLoads % WAVES;  // wavefronts with one more
  constexpr int kRowLoads = MR;                 // 2 rows of 512 bytes each
  static_assert((kMine + 1 + kRowLoads) * (STAGES - 1) <= 63, "vmcnt range");
  const int scale_row = scale_pitch(p.k);
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15;
  const int quad = lane >> 4;
  const int32_t n0 = static_cast<int32_t>(blockIdx.x) * 16 * NT;
  unsigned char *scales = smem + STAGES * kStage;
  const uint32_t lds0 = static_cast<uint32_t>(
      reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) unsigned char *)smem));
  const bool extra = wave < kExtra;

  // Piece i of row r at i ^ r, as above.
  const uint8_t *weight[kMine + 1];
  const int weight_piece = (lane & 7) ^ (lane >> 3);
#pragma unroll
  for (int i = 0; i <= kMine; ++i)
    weight[i] = p.weight +
                static_cast<int64_t>(min(n0 + 8 * (wave + WAVES * i) + (lane >> 3), p.n - 1)) * p.weight_stride;
  const T *x[kRowLoads];
  int row_piece[kRowLoads];
#pragma unroll
  for (int i = 0; i < kRowLoads; ++i) {
    const int row = 2 * (wave + WAVES * i) + (lane >> 5);
    x[i] = static_cast<const T *>(p.x) + static_cast<int64_t>(min(row, p.m - 1)) * p.x_stride;
    row_piece[i] = (lane & 31) ^ (row & 15);
  }
  auto load_weight = [&](int i, int32_t code, int stage) __attribute__((always_inline)) {
    load_lds16<true>(weight[i] + code,
                     __builtin_amdgcn_readfirstlane(lds0 + stage * kStage + (wave + WAVES * i) * 1024));
  };
  auto load = [&](int32_t base, int stage) __attribute__((always_inline)) {
    const int32_t code = min(base / 2 + 16 * weight_piece, p.k / 2 - 16);
#pragma unroll
    for (int i = 0; i < kMine; ++i) load_weight(i, code, stage);
    if (kExtra && extra) load_weight(kMine, code, stage);
#pragma unroll
    for (int i = 0; i < kRowLoads; ++i)
      load_lds16(x[i] + min(base + 8 * row_piece[i], p.k - 8),
                 __builtin_amdgcn_readfirstlane(lds0 + stage * kStage + kWeightBytes + (wave + WAVES * i) * 1024));
  };

  f32x4 acc[MR][NT];
#pragma unroll
  for (int r = 0; r < MR; ++r)
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[r][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  // This wavefront's products of a chunk: step `s` of group `piece`.
  const int piece = 4 * (wave / 4) + quad;
  const int s = wave % 4;

  // The chunk at `base`, FLIGHT chunks having been issued behind it; then one
  // more, at `next`, into the buffer of the chunk before.
  auto multiply = [&](auto flight, int32_t base, int32_t panel, int stage, int32_t next) {
    constexpr int kFlight = decltype(flight)::value;
    if (kExtra && extra)
      asm volatile("s_waitcnt vmcnt(%0)" : : "n"((kMine + 1 + kRowLoads) * kFlight) : "memory");
    else
      asm volatile("s_waitcnt vmcnt(%0)" : : "n"((kMine + kRowLoads) * kFlight) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" : : : "memory");
    if (next >= 0) load(next, stage == 0 ? STAGES - 1 : stage - 1);
    const unsigned char *at = smem + stage * kStage;
    uint32_t codes[NT], exponent[NT];
    V rows[MR];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      codes[t] = *reinterpret_cast<const uint32_t *>(at + (16 * t + col) * 128 + 16 * (piece ^ (col & 7)) + 4 * s);
      exponent[t] = scales[(16 * t + col) * scale_row + (base - panel) / 32 + piece];
    }
#pragma unroll
    for (int r = 0; r < MR; ++r)
      rows[r] = *reinterpret_cast<const V *>(at + kWeightBytes + (16 * r + col) * 512 + 16 * ((4 * piece + s) ^ col));
    asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
    if (base + kChunk > p.k && base + 32 * piece >= p.k) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        codes[t] = 0;
        exponent[t] = 127;
      }
#pragma unroll
      for (int r = 0; r < MR; ++r) rows[r] = V{0, 0, 0, 0, 0, 0, 0, 0};
    }
    if constexpr (__is_same(T, _Float16)) {
      bool wide = false;
#pragma unroll
      for (int t = 0; t < NT; ++t) wide |= exponent[t] - (127 - 13) > 26;
      if (__any(wide)) {
#pragma unroll
        for (int r = 0; r < MR; ++r) {
          bf16x8 high, low;
          split(rows[r], high, low);
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            asm volatile("" : "+v"(codes[t]));  // decoded again: the decoded weights would not fit beside the sums
            const bf16x8 a = Operand<__bf16>::decode(codes[t], __builtin_bit_cast(float, exponent[t] << 23));
            acc[r][t] = Operand<__bf16>::mfma(a, high, acc[r][t]);
            acc[r][t] = Operand<__bf16>::mfma(a, low, acc[r][t]);
          }
        }
        return;
      }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const V a = Operand<T>::decode(codes[t], __builtin_bit_cast(float, exponent[t] << 23));
#pragma unroll
      for (int r = 0; r < MR; ++r) acc[r][t] = Operand<T>::mfma(a, rows[r], acc[r][t]);
    }
  };

  for (int32_t panel = 0; panel < p.k; panel += kPanel) {
    const int32_t end = min(panel + kPanel, p.k);
    const int32_t chunks = (end - panel + kChunk - 1) / kChunk;
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i)
      if (i < chunks) load(panel + i * kChunk, i);
    load_scales<NT>(p, n0, panel, end, scales, scale_row);
    __syncthreads();
    int32_t c = 0;
    int stage = 0;
    auto step = [&](auto flight, bool more) {
      multiply(flight, panel + c * kChunk, panel, stage, more ? panel + (c + STAGES - 1) * kChunk : -1);
      stage = stage + 1 == STAGES ? 0 : stage + 1;
      ++c;
    };
    while (c + STAGES - 1 < chunks) step(std::integral_constant<int, STAGES - 2>{}, true);
    if constexpr (STAGES >= 3)
      if (chunks - c >= 2) step(std::integral_constant<int, 1>{}, false);
    if (chunks - c >= 1) step(std::integral_constant<int, 0>{}, false);
    __syncthreads();  // the panel's scales and the ring are done with
  }

  // The upper four wavefronts' sums go to the lower ones.
  f32x4 *sums = reinterpret_cast<f32x4 *>(smem);  // [4][MR][NT][64]
  f32x4 *mine = sums + wave % 4 * MR * NT * 64 + lane;
  if (wave >= 4) {
#pragma unroll
    for (int r = 0; r < MR; ++r)
#pragma unroll
      for (int t = 0; t < NT; ++t) mine[(r * NT + t) * 64] = acc[r][t];
  }
  __syncthreads();
  if (wave < 4) {
#pragma unroll
    for (int r = 0; r < MR; ++r)
#pragma unroll
      for (int t = 0; t < NT; ++t) mine[(r * NT + t) * 64] += acc[r][t];
  }
  __syncthreads();
  join<T, MR, NT>(p, sums, 4, 0, n0);
}

// Raise a kernel's dynamic LDS limit once per device (a failure shows up as a
// launch error).
template <auto KERNEL>
void raise_lds(size_t lds) {
  if (lds <= 64 * 1024) return;
  constexpr int kMaxDevices = 64;
  static std::atomic<bool> raised[kMaxDevices];
  int device = 0;
  if (hipGetDevice(&device) == hipSuccess && device >= 0 && device < kMaxDevices &&
      !raised[device].load(std::memory_order_acquire)) {
    if (hipFuncSetAttribute(reinterpret_cast<const void *>(KERNEL), hipFuncAttributeMaxDynamicSharedMemorySize,
                            160 * 1024) == hipSuccess)
      raised[device].store(true, std::memory_order_release);
  }
}

template <typename T, int XR, int NT>
int32_t launch_linear(LinearParams p, int waves, hipStream_t stream) {
  constexpr int stage = 1024 * (2 * NT + XR / 2);
  auto kernel = linear_mxfp4_kernel<T, XR, NT>;
  const size_t ring = static_cast<size_t>(waves) * ring_stages(stage) * stage + 16 * NT * scale_pitch(p.k) + 8;
  const size_t sums = static_cast<size_t>(waves) * NT * 64 * sizeof(f32x4);
  const size_t lds = ring > sums ? ring : sums;
  raise_lds<linear_mxfp4_kernel<T, XR, NT>>(lds);
  p.column_tiles = (p.n + 16 * NT - 1) / (16 * NT);
  p.row_blocks = (p.m + 15) / 16;
  const unsigned grid = static_cast<unsigned>((p.column_tiles + kXcds - 1) / kXcds * kXcds) * p.row_blocks;
  hipLaunchKernelGGL(kernel, dim3(grid), dim3(64 * waves), lds, stream, p);
  return check_launch("linear_mxfp4");
}

template <typename T, int XR>
int32_t launch_columns(const LinearParams &p, int tiles, int waves, hipStream_t stream) {
  switch (tiles) {
    case 1: return launch_linear<T, XR, 1>(p, waves, stream);
    case 2: return launch_linear<T, XR, 2>(p, waves, stream);
    case 3: return launch_linear<T, XR, 3>(p, waves, stream);
    default: return launch_linear<T, XR, 4>(p, waves, stream);
  }
}

// Columns of a tile (16 NT) and wavefronts of a workgroup.  A compute unit
// takes lines at about 53 B/ns whatever they hold, so the tile with the fewest
// bytes per unit wins: 16 NT weight rows and 16 rows of x (or as many as there
// are) for each round of 256 workgroups, partial rounds counting only where a
// third one follows.  Up to 256 workgroups have a unit each and take eight
// wavefronts, more take four, none more than there are chunks.  Measured, best
// of NT 1 to 4 with 2, 4 and 8 wavefronts against the choice (us): 1 row of
// 2048 x 5632 5.3 / 5.3, 8 of 28672 x 4096 15.6 / 16.6, 16 of 32000 x 2048
// 11.8 / 11.8, 16 of 4096 x 14336 15.0 / 15.0, 32 of 11264 x 2048 8.5 / 8.5,
// 64 of 2048 x 2048 5.2 / 5.2, 64 of 4096 x 4096 10.3 / 10.4.
constexpr int64_t kUnits = 256;

void choose_tile(const LinearParams &p, int loaded_rows, int &tiles, int &waves) {
  const int64_t blocks = (p.m + 15) / 16;
  int64_t best = 0;
  for (int nt = 1; nt <= 4; ++nt) {
    const int64_t grid = (p.n + 16 * nt - 1) / (16 * nt) * blocks;
    const int64_t rounds = grid <= 2 * kUnits ? (grid + kUnits - 1) / kUnits * kUnits : grid;
    const int64_t cost = rounds * (8 * nt + 2 * loaded_rows);  // bytes per column of K
    if (nt == 1 || cost < best) {
      best = cost;
      tiles = nt;
      waves = grid <= kUnits ? 8 : 4;
    }
  }
  while (waves > 1 && waves > (p.k + kChunk - 1) / kChunk) waves /= 2;
}

template <typename T, int XR>
int32_t launch_tile(const LinearParams &p, hipStream_t stream) {
  int tiles, waves;
  choose_tile(p, XR, tiles, waves);
  return launch_columns<T, XR>(p, tiles, waves, stream);
}

// All rows in a workgroup: above kWideColumns columns, where 256 workgroups of
// three operands' columns are filled, tiles as wide as one round of 256 needs.
// Three chunks in the ring, two where LDS does not hold three.  Measured against
// the tiles of 16 rows (us): 64 rows of 11264 x 2048 15.4 / 11.9, of 16384 x
// 4096 29.7 / 19.2, of 28672 x 4096 48.6 / 28.5, of 32000 x 2048 30.9 / 21.2,
// of 64000 x 1024 39.6 / 29.2, of 8704 x 14336 55.2 / 47.6; 40 rows of 28672 x
// 4096 39.9 / 24.0; 32 rows of 11264 x 2048 8.7 / 9.3, of 28672 x 4096 29.7 /
// 23.4; below, 64 rows of 4096 x 4096 10.4 / 10.6, of 2048 x 2048 5.4 / 7.0.
// 64 rows of 16384 x 4096 with 4 / 8 wavefronts 21.5 / 19.2.
constexpr int32_t kWideColumns = 8192;

template <typename T, int MR, int NT, int STAGES>
int32_t launch_wide_stages(const LinearParams &p, size_t lds, hipStream_t stream) {
  constexpr auto kernel = linear_mxfp4_rows_kernel<T, MR, NT, STAGES>;
  raise_lds<kernel>(lds);
  hipLaunchKernelGGL(kernel, dim3((p.n + 16 * NT - 1) / (16 * NT)), dim3(512), lds, stream, p);
  return check_launch("linear_mxfp4");
}

template <typename T, int MR, int NT>
int32_t launch_wide_tile(const LinearParams &p, hipStream_t stream) {
  constexpr size_t stage = 2048 * NT + 8192 * MR;
  const size_t scales = 16 * NT * scale_pitch(p.k) + 8;
  constexpr size_t sums = 4 * MR * NT * 64 * sizeof(f32x4);
  const auto lds = [&](size_t stages) { return stages * stage + scales > sums ? stages * stage + scales : sums; };
  if (lds(3) <= 160 * 1024) return launch_wide_stages<T, MR, NT, 3>(p, lds(3), stream);
  return launch_wide_stages<T, MR, NT, 2>(p, lds(2), stream);
}

// fp16 has the second path for weights past its range, with which the sums of
// more than 21 tiles do not stay in registers: wider calls then take tiles of
// four operands' columns (64 rows of 28672 x 4096 43.7 us).
template <typename T, int MR>
int32_t launch_wide(const LinearParams &p, hipStream_t stream) {
  constexpr int kMost = __is_same(T, _Float16) ? 21 / MR : 8;
  const int64_t width = (p.n + 16 * kUnits - 1) / (16 * kUnits);
  if (width == 3) return launch_wide_tile<T, MR, 3>(p, stream);
  if (width == 5) return launch_wide_tile<T, MR, 5>(p, stream);
  if constexpr (kMost >= 6)
    if (width == 6) return launch_wide_tile<T, MR, 6>(p, stream);
  if constexpr (kMost >= 7)
    if (width == 7) return launch_wide_tile<T, MR, 7>(p, stream);
  if constexpr (kMost >= 8)
    if (width >= 8) return launch_wide_tile<T, MR, 8>(p, stream);
  return launch_wide_tile<T, MR, 4>(p, stream);
}

template <typename T>
int32_t launch_rows(const LinearParams &p, hipStream_t stream) {
  if (p.m <= 2) return launch_tile<T, 2>(p, stream);
  if (p.m <= 4) return launch_tile<T, 4>(p, stream);
  if (p.m <= 8) return launch_tile<T, 8>(p, stream);
  if (p.m > 16 && p.n > kWideColumns) {
    if (p.m <= 32) return launch_wide<T, 2>(p, stream);
    if (p.m <= 48) return launch_wide<T, 3>(p, stream);
    return launch_wide<T, 4>(p, stream);
  }
  return launch_tile<T, 16>(p, stream);
}

// Bytes of codes from which weights that several row blocks read pass the
// caches by (64 rows of 2048 x 5632 cached 8.0 us, past 8.8; in these tiles, of
// 11264 x 2048 14.4 and 13.5); one row block always does (1 row of 2048 x 2048 4.0 and 3.8).
constexpr int64_t kCached = 8000000;

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
  if (n > 1 << 28 || k > 1 << 28) return fail(TF_ERROR_UNSUPPORTED, "linear_mxfp4 takes at most 2^28 columns and K");
  if (m == 0 || n == 0) return TF_SUCCESS;
  if (!x || !weight || !scales || !y) return fail(TF_ERROR_INVALID_ARGUMENT, "null tensor pointer");
  if (x_row_stride < k || weight_row_stride < k / 2 || scale_row_stride < k / 32 || y_row_stride < n ||
      (residual && residual_row_stride < n))
    return fail(TF_ERROR_INVALID_ARGUMENT, "row stride is shorter than the rows");
  if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(weight)) % 16 != 0 || x_row_stride % 8 != 0 ||
      weight_row_stride % 16 != 0)
    return fail(TF_ERROR_INVALID_ARGUMENT, "x and weight rows must be 16-byte aligned");
  const bool words = k % 128 == 0 && scale_row_stride % 4 == 0 && reinterpret_cast<uintptr_t>(scales) % 4 == 0;
  const LinearParams p{x,
                       static_cast<const uint8_t *>(weight),
                       static_cast<const uint8_t *>(scales),
                       residual,
                       y,
                       x_row_stride,
                       weight_row_stride,
                       scale_row_stride,
                       residual_row_stride,
                       y_row_stride,
                       m,
                       n,
                       k,
                       0,
                       0,
                       m <= 16 || static_cast<int64_t>(n) * k / 2 >= kCached,
                       words};
  hipStream_t s = static_cast<hipStream_t>(stream);
  return dtype == TF_DTYPE_FLOAT16 ? launch_rows<_Float16>(p, s) : launch_rows<__bf16>(p, s);
}
