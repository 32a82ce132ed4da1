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
// One workgroup per row, which it reads once: up to NV 16-byte vectors a thread
// stay in registers for every later look (longer rows are read again behind
// those).  The alternatives are ordered by value, equal values by index, a NaN
// above every number (as in tf_argmax_rows):
//
//  * the threads' maxima in 64 groups; the k-th largest group's is a bound t
//    that at least k elements reach and few pass (of 32,000 normal logits and
//    k = 20 about 25);
//  * elements above t go to a list in LDS, in any order; where they are fewer
//    than k, elements equal to t follow in the order of their index;
//  * each of the list counts those ahead of it: its place.
//
// Where the list overflows (the largest elements share few groups), t is
// raised to the k-th largest element itself, found bit by bit.
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

template <typename T, int NV, int THREADS>
__global__ void __launch_bounds__(THREADS)
token_logprobs_kernel(const T *__restrict__ logits, int64_t row_stride, int32_t columns,
                      const int64_t *__restrict__ tokens, float *__restrict__ logprobs, float *__restrict__ entropy,
                      float *__restrict__ top_logprobs, int64_t *__restrict__ top_tokens, int32_t top_k) {
  constexpr int VEC = 16 / sizeof(T);
  constexpr int kWaves = THREADS / 64;
  constexpr int kPass = THREADS * NV;             // vectors of a pass
  constexpr int kGroupLanes = THREADS / kGroups;  // 4 or 16
  struct alignas(16) Vec {
    T v[VEC];
  };
  __shared__ uint32_t group_keys[kGroups];
  __shared__ float wave_sums[kWaves], wave_weighted[kWaves];
  __shared__ int32_t wave_ones[kWaves], counts[2][kWaves];
  __shared__ uint32_t bound_key;
  __shared__ int32_t listed;
  __shared__ uint32_t list_key[kList];
  __shared__ int32_t list_index[kList];
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t r = blockIdx.x;
  const T *row = logits + r * row_stride;
  // Vector i holds columns VEC i - skew .. + VEC - 1: aligned whatever the row's
  // start is.  Those the row does not fill are loaded element by element.
  const int skew = static_cast<int>(reinterpret_cast<uintptr_t>(row) % 16 / sizeof(T));
  const int32_t vectors = (columns + skew + VEC - 1) / VEC;
  const T absent = from_float<T>(-__builtin_inff());
  auto load = [&](int32_t i) {
    Vec v;
    const int32_t c = i * VEC - skew;
    if (c >= 0 && c + VEC <= columns) {
      v = *reinterpret_cast<const Vec *>(row + c);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) v.v[e] = c + e >= 0 && c + e < columns ? row[c + e] : absent;
    }
    return v;
  };
  Vec held[NV];
#pragma unroll
  for (int u = 0; u < NV; ++u)
    if (u * THREADS + tid < vectors) held[u] = load(u * THREADS + tid);
  // f(value, column, whether it is one) for this thread's elements, in the
  // order of their column.
  auto visit = [&](auto f) {
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int32_t i = u * THREADS + tid;
      if (i >= vectors) continue;
#pragma unroll
      for (int e = 0; e < VEC; ++e) f(to_float(held[u].v[e]), i * VEC - skew + e);
    }
    for (int32_t i = kPass + tid; i < vectors; i += THREADS) {
      const Vec v = load(i);
#pragma unroll
      for (int e = 0; e < VEC; ++e) f(to_float(v.v[e]), i * VEC - skew + e);
    }
  };
  auto inside = [&](int32_t c) { return static_cast<uint32_t>(c) < static_cast<uint32_t>(columns); };

  int64_t token = -1;
  float given = __builtin_nanf("");
  if (tid == 0) {
    listed = 0;
    token = tokens[r];
    if (token >= 0 && token < columns) given = to_float(row[token]);
  }

  // The largest value (absent ones are -inf), as a key with NaN on top.
  float own = -__builtin_inff();
  bool nan = false;
  visit([&](float x, int32_t) {
    own = fmaxf(own, x);
    nan |= x != x;
  });
  const bool any = tid < vectors;
  const uint32_t own_key = !any ? 0u : nan ? 0xffffffffu : order_key(own);
  uint32_t key = own_key;
  float top = own;
#pragma unroll
  for (int offset = 1; offset < kGroupLanes; offset <<= 1)
    key = max(key, static_cast<uint32_t>(__shfl_xor(static_cast<int>(key), offset, 64)));
  if (lane % kGroupLanes == 0) group_keys[tid / kGroupLanes] = key;
  top = wave_max(top);
  if (lane == 0) wave_sums[wave] = top;
  __syncthreads();
  float m = wave_sums[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) m = fmaxf(m, wave_sums[w]);
  if (top_k > 0) {
    // The groups with fewer than top_k ahead of them, equal ones in order; each
    // wavefront looks at its own.
    const uint32_t mine = group_keys[lane];
    constexpr int kOwn = 64 / kGroupLanes;
#pragma unroll
    for (int g = 0; g < kOwn; ++g) {
      const int at = wave * kOwn + g;
      const uint32_t one = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(mine), at));
      const unsigned long long above = __ballot(mine > one), same = __ballot(mine == one);
      const int ahead = __popcll(above) + __popcll(same & ((1ull << at) - 1));
      if (ahead == top_k - 1 && lane == 0) bound_key = one;
    }
  }

  float sum = 0.f, weighted = 0.f;
  int32_t ones = 0;
  if (own == m) {
    visit([&](float x, int32_t c) {
      const float d = x - m;
      const float e = __expf(d);
      ones += d == 0.f && inside(c);
      sum += d == 0.f ? 0.f : e;
      weighted += e == 0.f ? 0.f : d * e;
    });
  } else {
    visit([&](float x, int32_t) {
      const float d = x - m;
      const float e = __expf(d);
      sum += e;
      weighted += e == 0.f ? 0.f : d * e;
    });
  }
  sum = wave_sum(sum);
  weighted = wave_sum(weighted);
#pragma unroll
  for (int offset = 32; offset > 0; offset >>= 1) ones += __shfl_xor(ones, offset, 64);
  __syncthreads();  // the maxima have been read
  if (lane == 0) {
    wave_sums[wave] = sum;
    wave_weighted[wave] = weighted;
    wave_ones[wave] = ones;
  }
  __syncthreads();
  sum = weighted = 0.f;
  ones = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    sum += wave_sums[w];
    weighted += wave_weighted[w];
    ones += wave_ones[w];
  }
  const float log_sum = ones == 1 ? log1pf(sum) : logf(static_cast<float>(ones) + sum);
  if (tid == 0) {
    logprobs[r] = (given - m) - log_sum;
    entropy[r] = log_sum - weighted / (static_cast<float>(ones) + sum);
  }
  if (top_k == 0) return;

  uint32_t bound = bound_key;
  auto list_above = [&] {
    if (own_key > bound)
      visit([&](float x, int32_t c) {
        if (!inside(c)) return;
        const uint32_t k = order_key(x);
        if (k <= bound) return;
        const int32_t at = atomicAdd(&listed, 1);
        if (at < kList) {
          list_key[at] = k;
          list_index[at] = c;
        }
      });
    __syncthreads();
    return listed;
  };
  int32_t above = list_above();
  if (above > kList) {
    // The k-th largest key, from its highest bit down.
    uint32_t found = 0;
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t trial = found | 1u << bit;
      int32_t mine = 0;
      if (own_key >= trial) visit([&](float x, int32_t c) { mine += inside(c) && order_key(x) >= trial; });
#pragma unroll
      for (int offset = 32; offset > 0; offset >>= 1) mine += __shfl_xor(mine, offset, 64);
      if (lane == 0) counts[bit & 1][wave] = mine;
      __syncthreads();
      int32_t all = 0;
      for (int w = 0; w < kWaves; ++w) all += counts[bit & 1][w];
      if (all >= top_k) found = trial;
    }
    bound = found;
    __syncthreads();
    if (tid == 0) listed = 0;
    __syncthreads();
    above = list_above();
  }
  // Elements equal to the bound, by index, up to top_k.
  if (above < top_k) {
    int32_t have = above;
    for (int32_t first = 0; first < vectors && have < top_k; first += THREADS) {
      const int32_t i = first + tid;
      uint32_t hits = 0;
      if (i < vectors && own_key >= bound) {
        Vec v;
        bool kept = false;
#pragma unroll
        for (int u = 0; u < NV; ++u)
          if (first == u * THREADS) {
            v = held[u];
            kept = true;
          }
        if (!kept) v = load(i);
#pragma unroll
        for (int e = 0; e < VEC; ++e)
          hits |= (inside(i * VEC - skew + e) && order_key(to_float(v.v[e])) == bound ? 1u : 0u) << e;
      }
      const int32_t mine = __popc(hits);
      int32_t before = 0, wave_total = 0;  // equal elements of earlier lanes, and of the wavefront
#pragma unroll
      for (int e = 1; e <= VEC; e <<= 1) {
        const unsigned long long with = __ballot(mine & e);
        before += e * __popcll(with & ((1ull << lane) - 1));
        wave_total += e * __popcll(with);
      }
      const int buffer = first / THREADS & 1;
      if (lane == 0) counts[buffer][wave] = wave_total;
      __syncthreads();
      int32_t at = have + before;
      for (int w = 0; w < kWaves; ++w) {
        if (w < wave) at += counts[buffer][w];
        have += counts[buffer][w];
      }
      for (int e = 0; e < VEC; ++e)
        if (hits >> e & 1) {
          if (at < top_k) {
            list_key[at] = bound;
            list_index[at] = i * VEC - skew + e;
          }
          ++at;
        }
    }
    __syncthreads();
    above = top_k;
  }
  for (int32_t c = tid; c < above; c += THREADS) {
    const uint32_t k = list_key[c];
    const int32_t index = list_index[c];
    int32_t ahead = 0;
    for (int32_t o = 0; o < above; ++o) ahead += list_key[o] > k || (list_key[o] == k && list_index[o] < index);
    if (ahead < top_k) {
      top_tokens[r * top_k + ahead] = index;
      top_logprobs[r * top_k + ahead] = (key_value(k) - m) - log_sum;
    }
  }
}

template <typename T>
struct Rows {
  const T *logits;
  int64_t row_stride;
  int32_t rows, columns;
  const int64_t *tokens;
  float *logprobs, *entropy, *top_logprobs;
  int64_t *top_tokens;
  int32_t top_k;

  template <int NV, int THREADS>
  void launch(hipStream_t stream) const {
    hipLaunchKernelGGL((token_logprobs_kernel<T, NV, THREADS>), dim3(static_cast<unsigned>(rows)), dim3(THREADS), 0,
                       stream, logits, row_stride, columns, tokens, logprobs, entropy, top_logprobs, top_tokens, top_k);
  }
  template <int THREADS>
  void launch(int nv, hipStream_t stream) const {
    switch (nv) {
      case 1: return launch<1, THREADS>(stream);
      case 2: return launch<2, THREADS>(stream);
      case 4: return launch<4, THREADS>(stream);
      case 8: return launch<8, THREADS>(stream);
      default: return launch<16, THREADS>(stream);
    }
  }
};

// Vectors a thread holds: the fewest of 1, 2, 4, 8, 16 for the row.
inline int held_vectors(int64_t vectors, int threads) {
  int nv = 1;
  while (nv < 16 && static_cast<int64_t>(nv) * threads < vectors) nv *= 2;
  return nv;
}

template <typename T>
void launch_logprobs(const void *logits, int64_t row_stride, int32_t rows, int32_t columns, const int64_t *tokens,
                     float *logprobs, float *entropy, float *top_logprobs, int64_t *top_tokens, int32_t top_k,
                     hipStream_t stream) {
  const Rows<T> all{static_cast<const T *>(logits), row_stride, rows, columns, tokens, logprobs, entropy,
                    top_logprobs, top_tokens, top_k};
  const int64_t vectors = static_cast<int64_t>(columns) * sizeof(T) / 16 + 2;
  if (vectors <= 1024)
    all.template launch<256>(held_vectors(vectors, 256), stream);
  else
    all.template launch<1024>(held_vectors(vectors, 1024), stream);
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
