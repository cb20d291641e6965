// The next token of each row of logits: temperature, top-k, top-p and min-p,
// from given Gumbel numbers (gfx950).
//
// Order: l descending, then index ascending, as a 64-bit key (the float's
// order-preserving integer, then the index complemented).  The tokens kept are
// a prefix of that order (top-k and top-p) cut by w >= min_p.  A prefix is
// found as the smallest key that is still in, by bisection over the key's
// bits: each step sums, over the tokens whose key is not below the middle, one
// (top-k) or w (top-p).
#include "pkda_common.h"
#include "serve/pkda_serve_gfx950.h"

namespace pkda {
namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;

struct SampleParams {
  const void* logits;
  int64_t logits_stride;
  const float* noise;
  int64_t noise_stride;
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  float temperature_all;
  int top_k_all;
  float top_p_all, min_p_all;
  int32_t* token;
  float* logprob;
  int vocab;
};

// Order-preserving integer of a float (-0 as +0); 0 for what is never taken
// (NaN and -inf), +inf as the largest finite number.
__device__ __forceinline__ uint32_t float_key(float x) {
  if (!(x > -INFINITY)) return 0;
  const uint32_t b = __float_as_uint(fminf(x, 3.402823466e38f) + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_float(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ uint64_t order_key(float x, int i) {
  const uint32_t k = float_key(x);
  return k == 0 ? 0 : (static_cast<uint64_t>(k) << 32) | static_cast<uint32_t>(~i);
}

// The block's sum / maximum, every thread getting it; the order is fixed.
template <typename V, typename F>
__device__ __forceinline__ V block_reduce(V v, V* lds, F f) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v = f(v, __shfl_xor(v, o));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  V r = lds[0];
#pragma unroll
  for (int i = 1; i < kWaves; ++i) r = f(r, lds[i]);
  return r;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_kernel(SampleParams p) {
  __shared__ uint64_t s_key[kWaves];
  __shared__ double s_sum[kWaves];
  const int row = blockIdx.x;
  const T* l = static_cast<const T*>(p.logits) + row * p.logits_stride;
  const float* noise = p.noise + row * p.noise_stride;
  const auto max_key = [](uint64_t a, uint64_t b) { return a > b ? a : b; };
  const auto add = [](double a, double b) { return a + b; };

  uint64_t top = 0;
  for (int i = threadIdx.x; i < p.vocab; i += kThreads) top = max_key(top, order_key(io<T>::load(l + i), i));
  top = block_reduce(top, s_key, max_key);
  if (top == 0) {
    if (threadIdx.x == 0) {
      p.token[row] = -1;
      p.logprob[row] = -INFINITY;
    }
    return;
  }
  const float m = key_float(static_cast<uint32_t>(top >> 32));
  const float T_ = p.temperature ? p.temperature[row] : p.temperature_all;
  uint64_t best = top;  // the token's order key
  if (T_ > 0.f) {
    const int k = p.top_k ? p.top_k[row] : p.top_k_all;
    const float top_p = p.top_p ? p.top_p[row] : p.top_p_all;
    const float min_p = p.min_p ? p.min_p[row] : p.min_p_all;
    const auto z_of = [&](uint64_t key) { return (key_float(static_cast<uint32_t>(key >> 32)) - m) / T_; };
    // sum of f over the keys >= lo
    const auto total = [&](uint64_t lo, bool mass) {
      double s = 0.;
      for (int i = threadIdx.x; i < p.vocab; i += kThreads) {
        const uint64_t key = order_key(io<T>::load(l + i), i);
        if (key != 0 && key >= lo) s += mass ? (double)expf(z_of(key)) : 1.;
      }
      return block_reduce(s, s_sum, add);
    };
    // the smallest key whose predecessors (keys above it) sum to less than goal,
    // not below floor: the predecessors of a key fall as the key rises
    const auto cut = [&](uint64_t floor, double goal, bool mass) {
      uint64_t lo = floor, hi = top;  // the answer is in [lo, hi]
      while (lo < hi) {
        const uint64_t mid = lo + (hi - lo) / 2;
        if (total(mid + 1, mass) < goal) hi = mid;
        else lo = mid + 1;
      }
      return lo;
    };
    uint64_t low = 1;
    if (k > 0) low = cut(1, (double)k, false);
    if (top_p < 1.f) low = cut(low, (double)top_p * total(low, true), true);
    uint64_t won = 0;
    float score = -INFINITY;
    for (int i = threadIdx.x; i < p.vocab; i += kThreads) {
      const uint64_t key = order_key(io<T>::load(l + i), i);
      if (key == 0 || key < low) continue;
      const float z = z_of(key);
      if (!(expf(z) >= min_p)) continue;
      const float s = z + noise[i];
      if (s > score) {
        score = s;
        won = key;
      }
    }
    // the best score, then the lowest index
    uint64_t pick = won == 0 ? 0
                             : (static_cast<uint64_t>(float_key(score)) << 32) | static_cast<uint32_t>(won);
    pick = block_reduce(pick, s_key, max_key);
    if (pick != 0) best = static_cast<uint32_t>(pick);
  }
  const int token = static_cast<int>(~static_cast<uint32_t>(best));
  double sum = 0.;
  for (int i = threadIdx.x; i < p.vocab; i += kThreads) {
    const uint32_t key = float_key(io<T>::load(l + i));
    if (key != 0) sum += (double)expf(key_float(key) - m);
  }
  sum = block_reduce(sum, s_sum, add);
  if (threadIdx.x == 0) {
    p.token[row] = token;
    p.logprob[row] = key_float(float_key(io<T>::load(l + token))) - m - (float)log(sum);
  }
}

}  // namespace
}  // namespace pkda

extern "C" int pkda_sample(const pkda_sample_args* a, void* stream) {
  using namespace pkda;
  PKDA_REQUIRE(a != nullptr, PKDA_EINVAL, "null args");
  PKDA_REQUIRE(a->struct_size == (int32_t)sizeof(*a), PKDA_EINVAL, "pkda_sample_args size mismatch");
  PKDA_REQUIRE(a->dtype == PKDA_F32 || a->dtype == PKDA_BF16, PKDA_EUNSUPPORTED, "dtype %d", a->dtype);
  PKDA_REQUIRE(a->rows >= 0 && a->vocab >= 1 && a->vocab <= (1 << 24), PKDA_EINVAL, "rows %d, vocab %d (1 .. 2^24)",
               a->rows, a->vocab);
  if (a->rows == 0) return 0;
  PKDA_REQUIRE(a->logits && a->noise && a->token && a->logprob, PKDA_EINVAL, "null tensor");
  PKDA_REQUIRE(a->logits_stride >= 0 && a->noise_stride >= 0, PKDA_EINVAL, "strides");
  SampleParams p = {a->logits, a->logits_stride, a->noise, a->noise_stride, a->temperature, a->top_k, a->top_p,
                    a->min_p, a->temperature_all, a->top_k_all, a->top_p_all, a->min_p_all, a->token, a->logprob, a->vocab};
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (a->dtype == PKDA_BF16)
    hipLaunchKernelGGL((sample_kernel<bf16_t>), dim3((unsigned)a->rows), dim3(kThreads), 0, s, p);
  else
    hipLaunchKernelGGL((sample_kernel<float>), dim3((unsigned)a->rows), dim3(kThreads), 0, s, p);
  return launch_status("pkda_sample");
}
