// The next token of each row of logits: temperature, top-k, top-p and min-p,
// from given Gumbel numbers (gfx950).
//
// One workgroup of 16 waves a row.  A row of V logits is read from memory once
// and again from the caches; at 131,072 logits one operation on each costs a
// compute unit 0.85 us (an exp 3.4), so what bounds a row is the operations a
// logit: the passes below touch most logits with a comparison only.
//
// Order: l falling, then index rising, as a 64-bit key: the float's
// order-preserving integer, then the index complemented.  The kept tokens are
// a prefix of that order (top-k and top-p) cut by w >= min_p.
//
// top_k <= 1024: the k-th largest of the threads' 1024 maxima is no larger than
// the k-th largest logit, and few more than k logits reach it.  They are
// gathered, sorted in LDS, and every setting is applied to the sorted list.
// Otherwise the last key of the prefix is found by rounds of a histogram of 32
// bins (one column a thread: no conflicts, a fixed order of additions) over the
// interval of keys it must lie in -- of e^z for top-p, of ones for a large
// top-k -- until the interval's tokens fit a list to sort.  Bins divide the
// logits' range evenly at first, then the keys', then the indices of one value.
//
// Scores z + noise are formed as the definition says, z by IEEE division, so
// that the token does not depend on the path.  Sums over bins and lists are FP64.
#include "pkda_common.h"
#include "serve/pkda_serve_gfx950.h"

namespace pkda {
namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kList = 1024;  // tokens of a sorted list: one a thread
constexpr int kBins = 32;
constexpr float kMaxFloat = 3.402823466e38f;
constexpr uint32_t kMinKey = 0x00800000u;  // the key of -kMaxFloat

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

// A logit as the operator takes it: NaN as -inf (never taken), +inf as the
// largest finite number.
__device__ __forceinline__ float usable(float x) { return x > -INFINITY ? fminf(x, kMaxFloat) : -INFINITY; }
// Order-preserving integer of a usable logit (-0 as +0); 0 for -inf.
__device__ __forceinline__ uint32_t float_key(float x) {
  if (!(x > -INFINITY)) return 0;
  const uint32_t b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_float(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ uint64_t order_key(float x, int i) {
  const uint32_t k = float_key(x);
  return k == 0 ? 0 : (static_cast<uint64_t>(k) << 32) | static_cast<uint32_t>(~i);
}
__device__ __forceinline__ int key_index(uint64_t key) { return static_cast<int>(~static_cast<uint32_t>(key)); }

// 16 bytes of a row that begins anywhere.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_any __attribute__((aligned(2)));
template <typename T> struct Logits;
template <> struct Logits<float> {
  static constexpr int N = 4;
  static constexpr uint32_t none = 0xff800000u;  // -inf
  __device__ __forceinline__ static float get(const u32x4& v, int j) { return __uint_as_float(v[j]); }
};
template <> struct Logits<bf16_t> {
  static constexpr int N = 8;
  static constexpr uint32_t none = 0xff80ff80u;
  __device__ __forceinline__ static float get(const u32x4& v, int j) {
    return __uint_as_float(j & 1 ? v[j / 2] & 0xffff0000u : v[j / 2] << 16);
  }
};

// f(logit, index) for a thread's logits of the row; a logit that does not exist
// comes as -inf.  Four vectors are loaded before the first is used.
template <typename T, typename F>
__device__ __forceinline__ void each(const T* l, int vocab, F f) {
  using L = Logits<T>;
  constexpr int U = 4;
  const int vectors = vocab / L::N;
  const u32x4_any* v = reinterpret_cast<const u32x4_any*>(l);
  for (int c = threadIdx.x; c < vectors; c += U * kThreads) {
    u32x4 x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      x[u] = u32x4{L::none, L::none, L::none, L::none};
      if (u == 0 || c + u * kThreads < vectors) x[u] = v[c + u * kThreads];
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < L::N; ++j) f(usable(L::get(x[u], j)), (c + u * kThreads) * L::N + j);
  }
  const int rest = vectors * L::N + threadIdx.x;
  if (rest < vocab) f(usable(io<T>::load(l + rest)), rest);
}

// f(logit, noise, index) for a thread's logits of the row.
template <typename T, typename F>
__device__ __forceinline__ void each_with_noise(const T* l, const float* noise, int vocab, F f) {
  using L = Logits<T>;
  typedef float f32x4 __attribute__((ext_vector_type(4)));
  typedef f32x4 f32x4_any __attribute__((aligned(4)));
  constexpr int U = 2;
  const int vectors = vocab / L::N;
  const u32x4_any* v = reinterpret_cast<const u32x4_any*>(l);
  for (int c = threadIdx.x; c < vectors; c += U * kThreads) {
    u32x4 x[U];
    f32x4 g[U][L::N / 4];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = u == 0 || c + u * kThreads < vectors ? c + u * kThreads : c;  // the same again: no harm
      x[u] = v[at];
#pragma unroll
      for (int q = 0; q < L::N / 4; ++q) g[u][q] = *reinterpret_cast<const f32x4_any*>(noise + at * L::N + 4 * q);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u > 0 && c + u * kThreads >= vectors) continue;
#pragma unroll
      for (int j = 0; j < L::N; ++j) f(usable(L::get(x[u], j)), g[u][j / 4][j % 4], (c + u * kThreads) * L::N + j);
    }
  }
  const int rest = vectors * L::N + threadIdx.x;
  if (rest < vocab) f(usable(io<T>::load(l + rest)), noise[rest], rest);
}

struct Lds {
  union {
    float hist[kBins][kThreads];
    uint64_t list[kList];
    uint32_t maxima[kThreads];
  };
  double bins[kBins];
  double wave_d[kWaves];
  uint64_t wave_k[kWaves];
  float wave_f[kWaves];
  int count;
};

// The block's reduction, every thread getting it; the order is fixed.
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
__device__ __forceinline__ uint64_t max_key(uint64_t a, uint64_t b) { return a > b ? a : b; }

// The sum of what the threads before this one have, and of all.
__device__ __forceinline__ double block_scan(double v, double* lds, double& total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  double s = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double y = __shfl_up(s, o);
    if (lane >= o) s += y;
  }
  __syncthreads();
  if (lane == 63) lds[w] = s;
  __syncthreads();
  double before = 0.;
  total = 0.;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    if (i < w) before += lds[i];
    total += lds[i];
  }
  return before + (s - v);
}

// Sorts n (a power of two, at most one a thread) keys in LDS, falling.  Steps
// within a wave need no barrier between them beyond the wave's own order.
template <typename K>
__device__ __forceinline__ void block_sort(K* s, int n) {
  const int i = threadIdx.x;
  K mine = i < n ? s[i] : 0;
  for (int size = 2; size <= n; size <<= 1)
    for (int step = size >> 1; step; step >>= 1) {
      K other;
      if (step >= 64) {
        __syncthreads();
        if (i < n) s[i] = mine;
        __syncthreads();
        other = i < n ? s[i ^ step] : 0;
      } else {
        other = __shfl_xor(mine, step);
      }
      const bool larger = ((i & step) == 0) == ((i & size) == 0);  // this place takes the larger
      if ((other > mine) == larger && other != mine) mine = other;
    }
  __syncthreads();
  if (i < n) s[i] = mine;
  __syncthreads();
}

// Gathers the keys that f gives (0: none) of the row's logits into the list;
// returns how many there are (more than kList: the list is not complete).
template <typename T, typename F>
__device__ __forceinline__ int gather(const T* l, int vocab, Lds& lds, F f) {
  __syncthreads();
  if (threadIdx.x == 0) lds.count = 0;
  __syncthreads();
  each(l, vocab, [&](float x, int i) {
    const uint64_t key = f(x, i);
    if (key != 0) {
      const int at = atomicAdd(&lds.count, 1);
      if (at < kList) lds.list[at] = key;
    }
  });
  __syncthreads();
  return lds.count;
}
__device__ __forceinline__ void sort_list(Lds& lds, int n) {
  int size = 64;
  while (size < n) size <<= 1;
  if ((int)threadIdx.x >= n && (int)threadIdx.x < size) lds.list[threadIdx.x] = 0;
  __syncthreads();
  block_sort(lds.list, size);
}

struct Row {
  float m, temperature, c;  // the largest logit; e^z = 2^((l - m) c)
  __device__ __forceinline__ float z(float x) const { return (x - m) / temperature; }
  __device__ __forceinline__ float weight(float x) const { return exp2_fast((x - m) * c); }
};

// How a round divides its interval of keys into bins.
struct Bins {
  int by;  // 0: value, 1: key, 2: index
  float top, inv;
  uint32_t high;
  int shift;
  __device__ __forceinline__ int of_value(float x) const { return (int)fminf((top - x) * inv, kBins - 1.f); }
  __device__ __forceinline__ int of_key(uint32_t k) const {
    return by == 0 ? of_value(key_float(k)) : (int)((high - k) >> shift);
  }
  __device__ __forceinline__ int of(uint64_t key) const {
    return by == 2 ? (int)((high - (uint32_t)key) >> shift) : of_key((uint32_t)(key >> 32));
  }
};

// The smallest key k of [lo, hi] with f(k) (false, then true as k rises; f(hi)
// holds), by the whole wave.
template <typename F>
__device__ __forceinline__ uint32_t first_key(uint32_t lo, uint32_t hi, F f) {
  const uint32_t lane = threadIdx.x & 63;
  while (lo < hi) {
    const uint32_t step = (hi - lo) / 64 + 1;
    const uint64_t at = (uint64_t)lo + (uint64_t)lane * step;
    const uint64_t holds = __ballot(at >= hi || f((uint32_t)at));
    const int n = __builtin_ctzll(holds);  // 64 when none holds: above lane 63
    if (holds == 0) {
      lo = lo + 63 * step + 1;
    } else {
      const uint64_t h = (uint64_t)lo + (uint64_t)n * step;
      if (n > 0) lo = lo + (n - 1) * step + 1;
      hi = h < hi ? (uint32_t)h : hi;
      if (n == 0) lo = hi;
    }
  }
  return lo;
}

// The last key of the prefix of the keys >= low0 that holds the tokens before
// which they hold less than goal tokens (count) or goal of their weight (mass).
// A first round over the whole row adds its e^(l - m) to exps, if that is not
// done yet.
struct Exps {
  float sum;
  bool done;
  __device__ __forceinline__ void add(float x, float m) { sum += exp2_fast((x - m) * kLog2e); }
};
template <typename T>
__device__ __forceinline__ uint64_t last_key(const T* l, int vocab, const Row& row, uint64_t low0, bool mass, double goal,
                                             Lds& lds, Exps& exps) {
  uint64_t lo = low0, hi = ((uint64_t)float_key(row.m) << 32) | 0xffffffffu;
  double before = 0.;
  for (int round = 0;; ++round) {
    const uint32_t klo = max((uint32_t)(lo >> 32), kMinKey), khi = (uint32_t)(hi >> 32);
    Bins b;
    b.top = key_float(khi);
    b.inv = 0.f;
    uint32_t range;
    if (klo == khi) {
      b.by = 2;
      b.high = min((uint32_t)hi, 0xffffffffu);
      range = b.high - max((uint32_t)lo, (uint32_t)~(vocab - 1));
    } else if (round < 3) {
      b.by = 0;
      b.high = khi;
      // from the top in steps of half an e-fold; later the whole interval
      const float all = (b.top - key_float(klo)) * (1.f / kBins);
      const float width = round == 0 ? fminf(all, mass ? 0.5f * row.temperature : 0.5f) : all;
      b.inv = 1.f / fmaxf(width, 1e-30f);
      range = 0;
    } else {
      b.by = 1;
      b.high = khi;
      range = khi - klo;
    }
    b.shift = 0;
    while ((range >> b.shift) >= kBins) ++b.shift;

    __syncthreads();
#pragma unroll
    for (int i = 0; i < kBins; ++i) lds.hist[i][threadIdx.x] = 0.f;
    const float fhi = b.top, flo = key_float(klo);
    const bool whole = lo <= ((uint64_t)kMinKey << 32) && b.by == 0 && round == 0;
    const bool add = whole && !exps.done;
    each(l, vocab, [&](float x, int i) {
      if (whole) {  // every usable logit
        if (add) exps.add(x, row.m);
        if (x > -INFINITY) lds.hist[b.of_value(x)][threadIdx.x] += mass ? row.weight(x) : 1.f;
      } else if (x >= flo && x <= fhi) {
        const uint64_t key = order_key(x, i);
        if (key >= lo && key <= hi) lds.hist[b.of(key)][threadIdx.x] += mass ? row.weight(x) : 1.f;
      }
    });
    if (add) exps.done = true;
    __syncthreads();
    // the bins' sums: two a wave
#pragma unroll
    for (int q = 0; q < kBins / kWaves; ++q) {
      const int bin = q * kWaves + (threadIdx.x >> 6);
      double s = 0.;
#pragma unroll
      for (int i = 0; i < kThreads / 64; ++i) s += lds.hist[bin][i * 64 + (threadIdx.x & 63)];
#pragma unroll
      for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
      if ((threadIdx.x & 63) == 0) lds.bins[bin] = s;
    }
    __syncthreads();
    if (round == 0) {
      double total = 0.;
      for (int i = 0; i < kBins; ++i) total += lds.bins[i];
      if (mass) goal *= total;
      else if (total <= goal) return low0;
    }
    int bin = -1;
    double at = before;
    for (int i = 0; i < kBins; ++i) {
      const double s = lds.bins[i];
      if (s > 0.) {
        bin = i;
        before = at;
        if (at + s >= goal) break;
        at += s;
      }
    }
    if (bin < 0) return lo;  // weights that are all zero
    // the bin's keys
    uint64_t nlo, nhi;
    if (b.by == 2) {
      const uint32_t h = b.high - ((uint32_t)bin << b.shift);
      const uint64_t span = (1ull << b.shift) - 1;
      nhi = ((uint64_t)khi << 32) | h;
      nlo = ((uint64_t)khi << 32) | (h > span ? (uint32_t)(h - span) : 0u);
    } else {
      const uint32_t first = first_key(klo, khi, [&](uint32_t k) { return b.of_key(k) <= bin; });
      const uint32_t past = bin == 0 ? khi : first_key(klo, khi, [&](uint32_t k) { return b.of_key(k) < bin; }) - 1;
      nlo = (uint64_t)first << 32;
      nhi = ((uint64_t)past << 32) | 0xffffffffu;
    }
    lo = max_key(lo, nlo);
    hi = nhi < hi ? nhi : hi;
    const float glo = key_float(max((uint32_t)(lo >> 32), kMinKey)), ghi = key_float((uint32_t)(hi >> 32));
    const int n = gather(l, vocab, lds, [&](float x, int i) -> uint64_t {
      if (!(x >= glo && x <= ghi)) return 0;
      const uint64_t key = order_key(x, i);
      return key >= lo && key <= hi ? key : 0;
    });
    if (n > kList) continue;
    sort_list(lds, n);
    const uint64_t mine = (int)threadIdx.x < n ? lds.list[threadIdx.x] : 0;
    const double part = mine == 0 ? 0. : mass ? (double)row.weight(key_float((uint32_t)(mine >> 32))) : 1.;
    double total;
    const double prior = before + block_scan(part, lds.wave_d, total);
    // the list falls: the last kept key is the least
    const uint64_t kept = mine != 0 && (prior < goal || threadIdx.x == 0) ? ~mine : 0;
    return ~block_reduce(kept, lds.wave_k, max_key);
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_kernel(SampleParams p) {
  __shared__ Lds lds;
  const int r = blockIdx.x;
  const T* l = static_cast<const T*>(p.logits) + r * p.logits_stride;
  const float* noise = p.noise + r * p.noise_stride;
  Row row;
  row.temperature = p.temperature ? p.temperature[r] : p.temperature_all;
  int k = p.top_k ? p.top_k[r] : p.top_k_all;
  const float top_p = p.top_p ? p.top_p[r] : p.top_p_all;
  const float min_p = p.min_p ? p.min_p[r] : p.min_p_all;
  if (k >= p.vocab) k = 0;

  float mine = -INFINITY;
  each(l, p.vocab, [&](float x, int) { mine = fmaxf(mine, x); });
  row.m = block_reduce(mine, lds.wave_f, [](float a, float b) { return fmaxf(a, b); });
  if (!(row.m > -INFINITY)) {
    if (threadIdx.x == 0) {
      p.token[r] = -1;
      p.logprob[r] = -INFINITY;
    }
    return;
  }
  row.c = fminf(kLog2e / row.temperature, kMaxFloat);
  Exps exps = {0.f, false};

  uint64_t pick = 0;  // the best score's key, then its token's index complemented
  const auto score = [&](float x, float g, int i) {
    const float s = row.z(x) + g;
    if (s > -INFINITY) pick = max_key(pick, ((uint64_t)float_key(fminf(s, kMaxFloat)) << 32) | (uint32_t)~i);
  };
  const auto likely = [&](float x) { return min_p <= 0.f || expf(row.z(x)) >= min_p; };

  if (row.temperature > 0.f) {
    bool done = false;
    if (k > 0 && k <= kList) {
      lds.maxima[threadIdx.x] = float_key(mine);
      __syncthreads();
      block_sort(lds.maxima, kThreads);
      const float least = key_float(max(lds.maxima[k - 1], kMinKey));
      const int n = gather(l, p.vocab, lds, [&](float x, int i) -> uint64_t {
        exps.add(x, row.m);
        return x >= least ? order_key(x, i) : 0;
      });
      exps.done = true;
      if (n <= kList) {
        sort_list(lds, n);
        const uint64_t key = (int)threadIdx.x < min(n, k) ? lds.list[threadIdx.x] : 0;
        const float x = key_float((uint32_t)(key >> 32));
        bool keep = key != 0;
        if (top_p < 1.f) {
          double total;
          const double before = block_scan(keep ? (double)row.weight(x) : 0., lds.wave_d, total);
          keep = keep && (before < (double)top_p * total || threadIdx.x == 0);
        }
        if (keep && likely(x)) score(x, noise[key_index(key)], key_index(key));
        done = true;
      }
    }
    if (!done) {
      uint64_t low = 1;
      if (k > 0) low = last_key(l, p.vocab, row, low, false, (double)k, lds, exps);
      if (top_p < 1.f) low = last_key(l, p.vocab, row, low, true, (double)top_p, lds, exps);
      if (low == 1 && min_p <= 0.f && exps.done) {
        each_with_noise(l, noise, p.vocab, score);
      } else if (low == 1 && min_p <= 0.f) {
        each_with_noise(l, noise, p.vocab, [&](float x, float g, int i) {
          exps.add(x, row.m);
          score(x, g, i);
        });
      } else {
        // what a logit must reach: the prefix's last value, and min_p's but for rounding
        float least = key_float(max((uint32_t)(low >> 32), kMinKey));
        if (min_p > 0.f) {
          const float d = row.temperature * logf(min_p);
          least = fmaxf(least, row.m + d - 1e-5f * (fabsf(row.m) + fabsf(d) + row.temperature));
        }
        const auto take = [&](float x, int i) {
          if (x >= least && order_key(x, i) >= low && likely(x)) score(x, noise[i], i);
        };
        if (exps.done)
          each(l, p.vocab, take);
        else
          each(l, p.vocab, [&](float x, int i) {
            exps.add(x, row.m);
            take(x, i);
          });
      }
      exps.done = true;
    }
    pick = block_reduce(pick, lds.wave_k, max_key);
  }
  if (pick == 0) {  // the first of the order: greedy, or noise that nothing wins
    each(l, p.vocab, [&](float x, int i) {
      if (!exps.done) exps.add(x, row.m);
      if (x == row.m) pick = max_key(pick, (1ull << 32) | (uint32_t)~i);
    });
    pick = block_reduce(pick, lds.wave_k, max_key);
  }
  const double total = block_reduce((double)exps.sum, lds.wave_d, [](double a, double b) { return a + b; });
  if (threadIdx.x == 0) {
    const int token = key_index(pick);
    p.token[r] = token;
    p.logprob[r] = (usable(io<T>::load(l + token)) - row.m) - (float)log(total);
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
                    a->min_p, a->temperature_all, a->top_k_all, a->top_p_all, a->min_p_all, a->token, a->logprob,
                    a->vocab};
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (a->dtype == PKDA_BF16)
    hipLaunchKernelGGL((sample_kernel<bf16_t>), dim3((unsigned)a->rows), dim3(kThreads), 0, s, p);
  else
    hipLaunchKernelGGL((sample_kernel<float>), dim3((unsigned)a->rows), dim3(kThreads), 0, s, p);
  return launch_status("pkda_sample");
}
