// Log probabilities of given tokens, the entropy of each row's distribution
// and its most likely tokens.
//
// For a row x: m = max x, S = sum exp(x - m);
//   log p(i) = (x[i] - m) - log S
//   H = log S - (sum (x - m) exp(x - m)) / S       (both terms >= 0)
// with the term of x = -inf zero.  The terms exp(0) = 1 of the maximum are
// counted, not summed: where it stands alone log S = log1p of the rest, so a
// sharp row keeps its small numbers.
//
// One workgroup per row, which it reads once: up to 16 vectors of 16 bytes a
// thread stay in registers for every later look (longer rows are read again
// behind those).  The alternatives are ordered by value, equal values by index, a NaN
// above every number (as in tf_argmax_rows):
//
//  * the threads' maxima in 64 groups, one a lane: the k-th largest group's is a
//    bound t that at least k elements reach and few pass (of 32,000 normal
//    logits and k = 20 about 25);
//  * the elements that reach t go to a list in LDS, in any order;
//  * each of the list counts those ahead of it: its place.
//
// Where the list overflows (ties, or a mask that leaves few groups) it takes the
// elements above t only, or, if they are still too many, above the k-th
// largest element, found bit by bit; then elements equal to t follow in the
// order of their index.
//
// Bound by vector work and latency beside the one read: 2048 rows of 32,000 bf16
// logits with 20 alternatives 48.5 us (2.7 TB/s), 64 rows with 5 9.4 us.
#include <type_traits>

#include "tf_common.hpp"

namespace tf {
namespace {

constexpr int32_t kMaxTop = 32;
constexpr int kGroups = 64;
constexpr int kList = 512;

// An unsigned integer above 0 that orders as the value does: -0 equals +0, NaN
// last; and back.
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t bits = __builtin_bit_cast(uint32_t, x + 0.f);
  return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t key) {
  if (key == 0xffffffffu) return __builtin_nanf("");
  return __builtin_bit_cast(float, key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// Combine over the 64 lanes by lane moves of the vector unit; every lane gets
// the result.
template <typename V, typename F>
__device__ __forceinline__ V over_wave(V v, F combine) {
  static_assert(sizeof(V) == 4, "32-bit values");
  auto moved = [&](auto ctrl) {
    const int bits = __builtin_bit_cast(int, v);
    const int other = __builtin_amdgcn_update_dpp(bits, bits, decltype(ctrl)::value, 0xf, 0xf, false);
    return __builtin_bit_cast(V, other);
  };
  v = combine(v, moved(std::integral_constant<int, 0xb1>{}));   // lane ^ 1
  v = combine(v, moved(std::integral_constant<int, 0x4e>{}));   // lane ^ 2
  v = combine(v, moved(std::integral_constant<int, 0x141>{}));  // the other quad of eight
  v = combine(v, moved(std::integral_constant<int, 0x140>{}));  // the other eight of sixteen
  uint32_t bits = __builtin_bit_cast(uint32_t, v);
  const auto rows = __builtin_amdgcn_permlane16_swap(bits, bits, false, false);
  const uint32_t even = rows[0], odd = rows[1];
  v = combine(__builtin_bit_cast(V, even), __builtin_bit_cast(V, odd));
  bits = __builtin_bit_cast(uint32_t, v);
  const auto halves = __builtin_amdgcn_permlane32_swap(bits, bits, false, false);
  const uint32_t low = halves[0], high = halves[1];
  return combine(__builtin_bit_cast(V, low), __builtin_bit_cast(V, high));
}

// NV vectors of VEC elements a thread in registers; NV = 0 (and VEC = 1, rows
// that 16-byte loads cannot take): none, every look reads the row.
template <typename T, int VEC, int NV, int THREADS>
__global__ void __launch_bounds__(THREADS) __attribute__((amdgpu_waves_per_eu(NV <= 4 ? 8 : 4)))
token_logprobs_kernel(const T *__restrict__ logits, int64_t row_stride, int32_t columns,
                      const int64_t *__restrict__ tokens, float *__restrict__ logprobs, float *__restrict__ entropy,
                      float *__restrict__ top_logprobs, int64_t *__restrict__ top_tokens, int32_t top_k) {
  struct alignas(sizeof(T) * VEC) Vec {
    T v[VEC];
  };
  constexpr int kWaves = THREADS / 64;
  __shared__ uint32_t group_keys[kGroups];
  __shared__ float wave_tops[kWaves], wave_sums[kWaves], wave_weighted[kWaves];
  __shared__ int32_t wave_ones[kWaves], counts[2][kWaves];
  __shared__ uint32_t bound_key;
  __shared__ int32_t listed;
  __shared__ uint32_t list_key[kList];
  __shared__ int32_t list_index[kList], places[kList];
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t r = blockIdx.x;
  const T *row = logits + r * row_stride;
  const Vec *vrow = reinterpret_cast<const Vec *>(row);
  const int32_t vectors = columns / VEC;
  // Columns behind the last whole vector, one a thread.
  const int32_t last = vectors * VEC + tid;
  const bool has_last = last < columns;
  Vec held[NV > 0 ? NV : 1];
#pragma unroll
  for (int u = 0; u < NV; ++u)
    if (u * THREADS + tid < vectors) held[u] = vrow[u * THREADS + tid];
  const T last_value = has_last ? row[last] : from_float<T>(0.f);
  // f(vector, its number) for this thread's, in order.  The packed vectors are
  // made new to the compiler each time, which otherwise keeps every element
  // unpacked in a register of its own.
  auto each_vector = [&](auto f) __attribute__((always_inline)) {
    if constexpr (NV > 0) {
#pragma unroll
      for (int u = 0; u < NV; ++u) {
        u32x4 bits = __builtin_bit_cast(u32x4, held[u]);
        asm volatile("" : "+v"(bits));
        held[u] = __builtin_bit_cast(Vec, bits);
      }
#pragma unroll
      for (int u = 0; u < NV; ++u)
        if (u * THREADS + tid < vectors) f(held[u], u * THREADS + tid);
    }
    for (int32_t i = NV * THREADS + tid; i < vectors; i += THREADS) f(vrow[i], i);
  };
  // f(value, column) for every element of this thread's.
  auto visit = [&](auto f) __attribute__((always_inline)) {
    each_vector([&](const Vec &v, int32_t i) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) f(to_float(v.v[e]), i * VEC + e);
    });
    if (has_last) f(to_float(last_value), last);
  };

  if (tid < kGroups) group_keys[tid] = 0;
  int64_t token = -1;
  float given = __builtin_nanf("");
  if (tid == 0) {
    listed = 0;
    token = tokens[r];
    if (token >= 0 && token < columns) given = to_float(row[token]);
  }

  float own = -__builtin_inff();
  visit([&](float x, int32_t) { own = fmaxf(own, x); });
  const auto larger = [](float a, float b) { return fmaxf(a, b); };
  const float wave_top = over_wave(own, larger);
  if (lane == 0) wave_tops[wave] = wave_top;
  __syncthreads();
  float m = wave_tops[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) m = fmaxf(m, wave_tops[w]);

  // In units of log2: t = (x - m) log2 e, e = 2^t, which is 0 from t = -150 on:
  // t is held above -200 in t e, so that x = -inf adds 0 to it.
  constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
  float sum = 0.f, weighted = 0.f;
  int32_t ones = 0;
  if (own == m) {
    visit([&](float x, int32_t) {
      const float t = (x - m) * kLog2e;
      const float e = __builtin_amdgcn_exp2f(t);
      ones += t == 0.f;
      sum += t == 0.f ? 0.f : e;
      weighted = __builtin_fmaf(fmaxf(t, -200.f), e, weighted);
    });
  } else {
    visit([&](float x, int32_t) {
      const float t = (x - m) * kLog2e;
      const float e = __builtin_amdgcn_exp2f(t);
      sum += e;
      weighted = __builtin_fmaf(fmaxf(t, -200.f), e, weighted);
    });
  }
  // The thread's largest element as a key, 0 without any.  A sum that is NaN
  // came from one, or from x - m of infinities.
  bool nan = sum != sum;
  if (__builtin_isinf(m)) {
    nan = false;
    visit([&](float x, int32_t) { nan |= x != x; });
  }
  const uint32_t own_key = tid >= vectors && !has_last ? 0u : nan ? 0xffffffffu : order_key(own);
  const auto add = [](auto a, auto b) { return a + b; };
  sum = over_wave(sum, add);
  weighted = over_wave(weighted, add);
  if (__any(ones != 0)) ones = over_wave(ones, add);
  if (lane == 0) {
    wave_sums[wave] = sum;
    wave_weighted[wave] = weighted;
    wave_ones[wave] = ones;
  }
  if (top_k > 0) atomicMax(&group_keys[lane], own_key);
  __syncthreads();
  sum = weighted = 0.f;
  ones = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    sum += wave_sums[w];
    weighted += wave_weighted[w];
    ones += wave_ones[w];
  }
  const float all = static_cast<float>(ones) + sum;
  const float log_sum = ones == 1 ? log1pf(sum) : logf(all);
  if (tid == 0) {
    logprobs[r] = (given - m) - log_sum;
    entropy[r] = log_sum - weighted * kLn2 / all;
  }
  if (top_k == 0) return;

  // The top_k-th of the groups, equal ones in order; each wavefront looks at its
  // share of them.
  {
    const uint32_t mine = group_keys[lane];
    constexpr int kOwn = kGroups / kWaves;
#pragma unroll
    for (int g = 0; g < kOwn; ++g) {
      const int at = wave * kOwn + g;
      const uint32_t one = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(mine), at));
      const unsigned long long above = __ballot(mine > one), same = __ballot(mine == one);
      const int ahead = __popcll(above) + __popcll(same & ((1ull << at) - 1));
      if (ahead == top_k - 1 && lane == 0) bound_key = one;
    }
  }
  __syncthreads();
  uint32_t bound = bound_key;
  // The elements whose key is at least `least` into the list; where they overflow
  // it, those above the bound, and then above the top_k-th largest.
  uint32_t least = bound;
  int32_t above;
  for (int attempt = 0;; ++attempt) {
    const float value = key_value(least);
    auto list = [&](float x, int32_t c) __attribute__((always_inline)) {
      const uint32_t k = order_key(x);
      if (k < least) return;
      const int32_t at = atomicAdd(&listed, 1);
      if (at < kList) {
        list_key[at] = k;
        list_index[at] = c;
      }
    };
    if (own_key >= least) {
      each_vector([&](const Vec &v, int32_t i) __attribute__((always_inline)) {
        float most = to_float(v.v[0]);
#pragma unroll
        for (int e = 1; e < VEC; ++e) most = fmaxf(most, to_float(v.v[e]));
        if (most < value && own_key != 0xffffffffu) return;
#pragma unroll
        for (int e = 0; e < VEC; ++e) list(to_float(v.v[e]), i * VEC + e);
      });
      if (has_last) list(to_float(last_value), last);
    }
    __syncthreads();
    above = listed;
    if (above <= kList) break;
    if (attempt == 1) {
      // The top_k-th largest key, from its highest bit down.
      uint32_t found = 0;
      for (int bit = 31; bit >= 0; --bit) {
        const uint32_t trial = found | 1u << bit;
        int32_t mine = 0;
        if (own_key >= trial) visit([&](float x, int32_t) { mine += order_key(x) >= trial; });
        mine = over_wave(mine, add);
        if (lane == 0) counts[bit & 1][wave] = mine;
        __syncthreads();
        int32_t reach = 0;
        for (int w = 0; w < kWaves; ++w) reach += counts[bit & 1][w];
        if (reach >= top_k) found = trial;
      }
      bound = found;
    }
    if (bound == 0xffffffffu) {  // NaN: nothing is above it
      least = 0;
      above = 0;
      break;
    }
    least = bound + 1;
    __syncthreads();
    if (tid == 0) listed = 0;
    __syncthreads();
  }
  if (least != bound && above < top_k) {
    // Elements equal to the bound, by index, up to top_k: whole vectors, a round
    // of the workgroup at a time, then the columns behind them.
    int32_t have = above;
    for (int32_t first = 0, round = 0; have < top_k && first < vectors + THREADS; first += THREADS, ++round) {
      const int32_t i = first + tid;
      uint32_t hits = 0;
      int32_t column = i * VEC;
      if (first >= vectors) {
        column = last;
        hits = has_last && order_key(to_float(last_value)) == bound;
      } else if (i < vectors && own_key >= bound) {
        Vec v = vrow[i];
#pragma unroll
        for (int e = 0; e < VEC; ++e) hits |= (order_key(to_float(v.v[e])) == bound ? 1u : 0u) << e;
      }
      const int32_t mine = __popc(hits);
      int32_t before = 0, wave_total = 0;  // equal elements of earlier lanes, and of the wavefront
#pragma unroll
      for (int e = 1; e <= VEC; e <<= 1) {
        const unsigned long long with = __ballot(mine & e);
        before += e * __popcll(with & ((1ull << lane) - 1));
        wave_total += e * __popcll(with);
      }
      if (lane == 0) counts[round & 1][wave] = wave_total;
      __syncthreads();
      int32_t at = have + before;
      for (int w = 0; w < kWaves; ++w) {
        if (w < wave) at += counts[round & 1][w];
        have += counts[round & 1][w];
      }
      for (int e = 0; e < VEC; ++e)
        if (hits >> e & 1) {
          if (at < top_k) {
            list_key[at] = bound;
            list_index[at] = column + e;
          }
          ++at;
        }
    }
    __syncthreads();
    above = top_k;
  }
  // Lanes take the list's elements, wavefronts the ones compared with.
  for (int32_t c = tid; c < above; c += THREADS) places[c] = 0;
  __syncthreads();
  for (int32_t c = lane; c < above; c += 64) {
    const uint32_t k = list_key[c];
    const int32_t index = list_index[c];
    int32_t ahead = 0;
    for (int32_t o = wave; o < above; o += kWaves)
      ahead += list_key[o] > k || (list_key[o] == k && list_index[o] < index);
    if (ahead) atomicAdd(&places[c], ahead);
  }
  __syncthreads();
  for (int32_t c = tid; c < above; c += THREADS) {
    const int32_t place = places[c];
    if (place >= top_k) continue;
    top_tokens[r * top_k + place] = list_index[c];
    top_logprobs[r * top_k + place] = (key_value(list_key[c]) - m) - log_sum;
  }
}

template <typename T>
struct Rows {
  static constexpr int VEC = 16 / sizeof(T);
  const T *logits;
  int64_t row_stride;
  int32_t rows, columns;
  const int64_t *tokens;
  float *logprobs, *entropy, *top_logprobs;
  int64_t *top_tokens;
  int32_t top_k;

  template <int V, int NV, int THREADS>
  void launch(hipStream_t stream) const {
    hipLaunchKernelGGL((token_logprobs_kernel<T, V, NV, THREADS>), dim3(static_cast<unsigned>(rows)), dim3(THREADS), 0,
                       stream, logits, row_stride, columns, tokens, logprobs, entropy, top_logprobs, top_tokens, top_k);
  }
  // With the fewest of 1, 2, 4, 8, 16 vectors a thread that hold the row.
  template <int THREADS>
  void launch(hipStream_t stream) const {
    const int64_t each = (columns / VEC + THREADS - 1) / THREADS;
    if (each <= 1) return launch<VEC, 1, THREADS>(stream);
    if (each <= 2) return launch<VEC, 2, THREADS>(stream);
    if (each <= 4) return launch<VEC, 4, THREADS>(stream);
    if (each <= 8) return launch<VEC, 8, THREADS>(stream);
    return launch<VEC, 16, THREADS>(stream);
  }
};

// Threads of a row: 256 up to 1024 vectors, 1024 above; 512 where a unit has
// several rows and 1024 threads of eight vectors would leave room for one (512
// x 32000 fp32 logits, 20 alternatives: 25.0 us with 1024, 21.3 with 512; 64 x
// 131072 bf16, a row a unit, 22.8 and 38.3).
constexpr int32_t kUnits = 256;

template <typename T>
void launch_logprobs(const void *logits, int64_t row_stride, int32_t rows, int32_t columns, const int64_t *tokens,
                     float *logprobs, float *entropy, float *top_logprobs, int64_t *top_tokens, int32_t top_k,
                     hipStream_t stream) {
  const Rows<T> all{static_cast<const T *>(logits), row_stride, rows, columns, tokens, logprobs, entropy,
                    top_logprobs, top_tokens, top_k};
  const bool whole = reinterpret_cast<uintptr_t>(logits) % 16 == 0 && row_stride % Rows<T>::VEC == 0;
  if (!whole)
    all.template launch<1, 0, 1024>(stream);
  else if (columns / Rows<T>::VEC <= 1024)
    all.template launch<256>(stream);
  else if (rows > kUnits && columns / Rows<T>::VEC > 4096 && columns / Rows<T>::VEC <= 8192)
    all.template launch<512>(stream);
  else
    all.template launch<1024>(stream);
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
  if (columns > 1 << 30) return fail(TF_ERROR_UNSUPPORTED, "log probabilities take at most 2^30 columns");
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
