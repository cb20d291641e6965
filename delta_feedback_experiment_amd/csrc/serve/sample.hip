// The next token of each row of logits: temperature, top-k, top-p and min-p,
// from given Gumbel numbers (gfx950).
//
// One workgroup of 16 waves a row.  A row is read from memory once and again
// from the caches: at 131,072 logits one operation on each costs a compute unit
// 0.85 us (an exp 3.4), so what bounds a row is the operations a logit.  A first
// pass takes each thread's maximum and its sum of e^l against that maximum
// (rescaled when it grows); most rows then need one pass of comparisons more.
//
// Order: l falling, then index rising, as a 64-bit key: the float's
// order-preserving integer, then the index complemented.  The kept tokens are
// a prefix of that order (top-k and top-p) cut by w >= min_p.
//
// top_k <= 1024: the k-th largest of the threads' 1024 maxima (its upper 16 bits)
// is no larger than the k-th largest logit, and few more than k logits reach it.
// They are gathered, sorted in LDS, and every setting is applied to the sorted
// list.
// Otherwise the prefix's last key is found by rounds of a histogram over the
// row (one column of bins a thread: no conflicts, a fixed order of additions) --
// of e^z for top-p, of ones for a large top-k -- each finer around the bin in
// which the prefix ends, until that bin's tokens are few enough to sort.  Bins
// divide the logits' range evenly at first, then the keys', then one value's
// indices.
//
// Scores z + noise are those of the definition, z correctly rounded, so that the
// token does not depend on the path.  A thread's own sums are FP32, or whole
// numbers over lists, whose order varies; sums over threads and bins are FP64.
//
// Measured, BF16, 256 rows of 131,072 normal logits times 3 (a row a compute
// unit; 67 MB read once are 17 us, with all the noise 42): greedy 17 us, top-k 50
// 29 to 32 by its logits, top-k 200 and top-p 0.9 35, min-p 0.05 27, no filter 45,
// top-p 0.5 53, 0.9 90, 0.99 109, top-k 5000 97; 4 rows of 50,304: 9 to 56.  What is left of a
// top-p row is one exponential and one column addition a logit, then some 20
// block-wide steps one after another.
#include "logits.h"

namespace pkda {
namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kList = 1024;              // tokens of a sorted list: one a thread
constexpr int kBins = 32, kFewBins = 8;  // of a round over the row, over a list: what LDS has room for
constexpr int kCandidates = 27136;       // tokens of an unsorted list: likewise
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
__device__ __forceinline__ float key_logit(uint64_t key) { return key_float(static_cast<uint32_t>(key >> 32)); }

// A row of logits and its noise.  odd: some logit is NaN or +inf, so that every
// vector is cleaned as it is read.
template <typename T> struct RowData {
  using L = Logits<T>;
  const T* l;
  const float* noise;
  int vocab;
  bool odd;

  __device__ __forceinline__ int vectors() const { return vocab / L::N; }
  __device__ __forceinline__ float one(int i) const {
    u32x4 v = {0, 0, 0, 0};
    if constexpr (sizeof(T) == 2) v[0] = l[i];
    else v[0] = __float_as_uint(l[i]);
    if (odd) L::clean(v);
    return L::get(v, 0);
  }
  // The thread's vectors c, c + kThreads, ...; those past the row as -inf.
  template <int U>
  __device__ __forceinline__ void load(u32x4 (&x)[U], int c) const {
    const u32x4_any* v = reinterpret_cast<const u32x4_any*>(l);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      x[u] = u32x4{L::none, L::none, L::none, L::none};
      if (u == 0 || c + u * kThreads < vectors()) x[u] = v[c + u * kThreads];
    }
    if (odd)
#pragma unroll
      for (int u = 0; u < U; ++u) L::clean(x[u]);
  }
  // f(four vectors, the first one's number) over the thread's vectors.  (The next
  // four on their way meanwhile: 18 -> 21 us a row of 131,072.)
  template <typename F>
  __device__ __forceinline__ void batches(F f) const {
    for (int c = threadIdx.x; c < vectors(); c += 4 * kThreads) {
      u32x4 x[4];
      load(x, c);
      f(x, c);
    }
  }
  // The logit past the last whole vector that is this thread's, or -1.
  __device__ __forceinline__ int rest() const {
    const int i = vectors() * L::N + threadIdx.x;
    return i < vocab ? i : -1;
  }
  // f(logit, index) for the thread's logits, those past the row as -inf.
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    batches([&](const u32x4 (&x)[4], int c) {
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int j = 0; j < L::N; ++j) f(L::get(x[u], j), (c + u * kThreads) * L::N + j);
    });
    const int i = rest();
    if (i >= 0) f(one(i), i);
  }
  // f(logit, logit): likewise two at a time
  template <typename F>
  __device__ __forceinline__ void each2(F f) const {
    batches([&](const u32x4 (&x)[4], int) {
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int j = 0; j < L::N; j += 2) f(L::get(x[u], j), L::get(x[u], j + 1));
    });
    const int i = rest();
    if (i >= 0) f(one(i), -INFINITY);
  }
  // f(logit, noise, index)
  template <typename F>
  __device__ __forceinline__ void each_with_noise(F f) const {
    constexpr int U = 2;
    for (int c = threadIdx.x; c < vectors(); c += U * kThreads) {
      u32x4 x[U];
      f32x4 g[U][L::N / 4];
      load(x, c);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int at = u == 0 || c + u * kThreads < vectors() ? c + u * kThreads : c;  // again: its logits are -inf
#pragma unroll
        for (int q = 0; q < L::N / 4; ++q) g[u][q] = *reinterpret_cast<const f32x4_any*>(noise + (int64_t)at * L::N + 4 * q);
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < L::N; ++j) f(L::get(x[u], j), g[u][j / 4][j % 4], (c + u * kThreads) * L::N + j);
    }
    const int i = rest();
    if (i >= 0) f(one(i), noise[i], i);
  }
};

struct Lds {
  union {
    float hist[kBins + 2][kThreads];
    struct {
      uint32_t candidates[kCandidates];  // indices
      uint32_t few[kFewBins + 2][kThreads];
    };
  };
  uint64_t list[kList];
  union {
    int ranks[4][kThreads / 4];
    int counts[2][16][kWaves];
  };
  double bins[64];
  double wave_d[kWaves];
  uint64_t wave_k[kWaves];
  float wave_f[kWaves];
  int count, listed;
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
__device__ __forceinline__ float max_float(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ double add_double(double a, double b) { return a + b; }

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

// Sorts n (a power of two, at most one a thread) keys in LDS, falling: a bitonic
// network, its steps inside a wave by lane exchange.
template <typename K>
__device__ __forceinline__ void block_sort(K* s, int n) {
  const int i = threadIdx.x;
  __syncthreads();
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
constexpr int kRanked = kThreads / 4;  // a list this short is sorted by ranks
__device__ __forceinline__ void sort_list(Lds& lds, int n) {
  if (n > kRanked) {
    int size = 2 * kRanked;
    while (size < n) size <<= 1;
    if ((int)threadIdx.x >= n && (int)threadIdx.x < size) lds.list[threadIdx.x] = 0;
    block_sort(lds.list, size);
    return;
  }
  // a key's rank is the number of larger ones (no two are equal): four threads
  // compare it with a quarter of the list each
  const int i = threadIdx.x % kRanked, part = threadIdx.x / kRanked;
  if ((int)threadIdx.x >= n && (int)threadIdx.x < kRanked) lds.list[threadIdx.x] = 0;
  __syncthreads();
  const uint64_t mine = lds.list[i];
  const int quarter = (n + 3) / 4;
  int rank = 0;
#pragma unroll 8
  for (int j = part * quarter; j < min(n, (part + 1) * quarter); ++j) rank += lds.list[j] > mine;
  lds.ranks[part][i] = rank;
  __syncthreads();
  if (part == 0 && i < n) lds.list[lds.ranks[0][i] + lds.ranks[1][i] + lds.ranks[2][i] + lds.ranks[3][i]] = mine;
  __syncthreads();
}

// A 16-bit number that at least k of the threads' reach (0 when fewer than k are
// above it): four rounds of four bits, each counting the threads that reach
// fifteen numbers.
__device__ __forceinline__ uint32_t reached_by(uint32_t mine, int k, Lds& lds) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  uint32_t found = 0;
  __syncthreads();
#pragma unroll
  for (int shift = 12; shift >= 0; shift -= 4) {
    int reach = 0;
#pragma unroll
    for (int d = 1; d < 16; ++d) {
      const int n = __popcll(__ballot(mine >= (found | (uint32_t)d << shift)));
      if (lane == d) reach = n;
    }
    int (&counts)[16][kWaves] = lds.counts[(shift >> 2) & 1];
    if (lane < 16) counts[lane][w] = reach;
    __syncthreads();
    int sum = 0;
    if (lane < 16)
#pragma unroll
      for (int i = 0; i < kWaves; ++i) sum += counts[lane][i];
    const uint64_t enough = __ballot(lane > 0 && lane < 16 && sum >= k);
    found |= (uint32_t)__popcll(enough) << shift;
  }
  return found;
}

// A place in a list of LDS for every active lane, one addition a wave; the
// places' order is no matter: lists are sorted, or searched for one maximum.
__device__ __forceinline__ int take_places(int* count) {
  const uint64_t active = __ballot(true);
  const int before = __builtin_amdgcn_mbcnt_hi((uint32_t)(active >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)active, 0));
  int at = 0;
  if (before == 0) at = atomicAdd(count, __popcll(active));
  return __builtin_amdgcn_readfirstlane(at) + before;
}
// The same within each wave, k / 16 of its threads, and the least of the waves'
// numbers: no counts to exchange, for a few more logits that reach it.
__device__ __forceinline__ uint32_t reached_by_waves(uint32_t mine, int k, Lds& lds) {
  const int need = (k + kWaves - 1) / kWaves;
  uint32_t found = 0;
#pragma unroll
  for (int bit = 15; bit >= 0; --bit) {
    const uint32_t t = found | 1u << bit;
    if (__popcll(__ballot(mine >= t)) >= need) found = t;
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds.wave_f[threadIdx.x >> 6] = (float)found;
  __syncthreads();
  float least = lds.wave_f[0];
#pragma unroll
  for (int i = 1; i < kWaves; ++i) least = fminf(least, lds.wave_f[i]);
  return (uint32_t)least;
}

// The indices of the logits that reach least, into the candidates; returns how
// many there are (more than kCandidates: the list is not complete).  Four
// vectors' comparisons make a lane's mask, one addition a wave the places of all.
template <typename T>
__device__ __forceinline__ int gather(const RowData<T>& row, float least, Lds& lds) {
  using L = Logits<T>;
  __syncthreads();
  if (threadIdx.x == 0) lds.count = 0;
  __syncthreads();
  row.batches([&](const u32x4 (&x)[4], int c) {
    uint32_t mask = 0;
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int j = 0; j < L::N; ++j) mask |= L::get(x[u], j) >= least ? 1u << (u * L::N + j) : 0u;
    const int n = __popc(mask);
    const uint64_t any = __ballot(n != 0);
    if (any == 0) return;
    int at = 0;
    if (__popcll(any) <= 8) {
      if (n != 0) at = atomicAdd(&lds.count, n);
      while (mask) {
        const int b = __builtin_ctz(mask);
        mask &= mask - 1;
        if (at < kCandidates) lds.candidates[at] = (c + b / L::N * kThreads) * L::N + b % L::N;
        ++at;
      }
      return;
    }
    // the lanes before this one have sum over bits b of 2^b times those whose n has it
    int before = 0, all = 0;
#pragma unroll
    for (int b = 0; b < 6; ++b) {
      const uint64_t has = __ballot((n >> b) & 1);
      before += (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(has >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)has, 0)) << b;
      all += __popcll(has) << b;
    }
    if (before == 0) {  // the first lanes: one of them, of the active ones, adds
      const uint64_t first = __ballot(true);
      if ((int)(threadIdx.x & 63) == __builtin_ctzll(first)) at = atomicAdd(&lds.count, all);
    }
    at = __builtin_amdgcn_readfirstlane(at) + before;
    while (mask) {
      const int b = __builtin_ctz(mask);
      mask &= mask - 1;
      if (at < kCandidates) lds.candidates[at] = (c + b / L::N * kThreads) * L::N + b % L::N;
      ++at;
    }
  });
  const int i = row.rest();
  if (i >= 0 && row.one(i) >= least) {
    const int at = take_places(&lds.count);
    if (at < kCandidates) lds.candidates[at] = i;
  }
  __syncthreads();
  return lds.count;
}

// A row's logits, or a list of them: f(logit, index).
template <typename T> struct Source {
  const RowData<T>& row;
  const uint32_t* list;  // nullptr: the row
  int n;
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    if (!list) {
      row.each(f);
      return;
    }
    constexpr int U = 8;
    for (int i = threadIdx.x; i < n; i += U * kThreads) {
      int at[U];
      float x[U];
#pragma unroll
      for (int u = 0; u < U; ++u) at[u] = i + u * kThreads < n ? (int)list[i + u * kThreads] : -1;
#pragma unroll
      for (int u = 0; u < U; ++u) x[u] = at[u] >= 0 ? row.one(at[u]) : 0.f;
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (at[u] >= 0) f(x[u], at[u]);
    }
  }
};

// What a row's softmax needs.
struct Scale {
  float m, temperature;  // the largest logit
  float c, from, shift;  // e^z = 2^((l - from) c + shift), c = log2 e / temperature
  float inv;             // 1 / temperature, or 0 where z takes the division itself
  __device__ __forceinline__ void init(float top, float t) {
    m = top;
    temperature = t;
    // above 0 also for an infinite temperature: -inf has the weight 0, not NaN, and
    // a finite logit one within 2^-21 of 1
    c = fmaxf(fminf(kLog2e / t, kMaxFloat), 0x1p-149f);
    // l c - m c in one operation: every weight of a row is off by one factor, the
    // rounding of m c, which must stay near 1
    const bool near = fabsf(m * c) <= 0x1p20f;
    from = near ? 0.f : m;
    shift = near ? -(m * c) : 0.f;
    inv = t >= 0x1p-20f && t <= 0x1p20f ? 1.f / t : 0.f;
  }
  __device__ __forceinline__ float weight(float x) const { return exp2_fast(__builtin_fmaf(x - from, c, shift)); }
  // (x - m) / temperature, correctly rounded: from the rounded reciprocal by two
  // corrections (P. Markstein, "Computation of elementary functions on the IBM
  // RISC System/6000 processor", 1990), five operations where a division has
  // eleven.
  __device__ __forceinline__ float z_fast(float x) const {
    const float d = x - m;
    float q = d * inv;
    q = __builtin_fmaf(__builtin_fmaf(-q, temperature, d), inv, q);
    return __builtin_fmaf(__builtin_fmaf(-q, temperature, d), inv, q);
  }
  // (the difference of two finite logits is finite)
  __device__ __forceinline__ float z(float x) const { return fmaxf(x - m, -kMaxFloat) / temperature; }
};

// How a round divides an interval of keys: rows 1 .. n, falling, exactly; row 0 is
// above the interval, row n + 1 below it (or, open, below the bins).
struct Bins {
  int n;
  int by;  // 0: value, 1: key, 2: index of one value
  bool open;
  float inv, top1, least, most;  // row = 1 + (most - x) inv
  uint32_t low, high, low_index, high_index;
  int shift;
  // within the interval
  __device__ __forceinline__ int of_near(float x) const {
    return (int)__builtin_amdgcn_fmed3f(__builtin_fmaf(-x, inv, top1), 1.f, (float)(open ? n + 1 : n));
  }
  __device__ __forceinline__ int of_value(float x) const { return x > most ? 0 : x < least ? n + 1 : of_near(x); }
  __device__ __forceinline__ int of_key(uint32_t k) const {
    return k > high ? 0 : k < low ? n + 1 : by == 0 ? of_near(key_float(k)) : 1 + (int)((high - k) >> shift);
  }
  __device__ __forceinline__ int of(uint64_t key) const {
    const uint32_t k = (uint32_t)(key >> 32), i = (uint32_t)key;
    if (by != 2 || k != high) return of_key(k);
    return i > high_index ? 0 : i < low_index ? n + 1 : 1 + (int)((high_index - i) >> shift);
  }
};

// The smallest key k of [lo, hi] with f(k) (false, then true as k rises; f(hi)
// holds), by every wave for itself: the 64 keys around a guess, else 64 keys a
// step over what is left.
template <typename F>
__device__ __forceinline__ uint32_t first_key(uint32_t lo, uint32_t hi, uint32_t guess, F f) {
  const uint32_t lane = threadIdx.x & 63;
  if (hi - lo > 64) {
    const uint32_t base = min(max(guess, lo + 32) - 32, hi - 63);
    const uint64_t holds = __ballot(f(base + lane));
    if (holds == 0) {
      lo = base + 63 + 1;
    } else {
      const int n = __builtin_ctzll(holds);
      if (n > 0 || base == lo) return base + n;
      hi = base;
    }
  }
  while (lo < hi) {
    const uint32_t step = (hi - lo) / 64 + 1;
    const uint64_t at = (uint64_t)lo + (uint64_t)lane * step;
    const uint64_t holds = __ballot(at >= hi || f((uint32_t)at));
    if (holds == 0) {  // above lane 63's
      lo = lo + 63 * step + 1;
      continue;
    }
    const int n = __builtin_ctzll(holds);
    const uint64_t h = (uint64_t)lo + (uint64_t)n * step;
    hi = h < hi ? (uint32_t)h : hi;
    lo = n == 0 ? hi : lo + (n - 1) * step + 1;
  }
  return lo;
}

// Where a prefix ends: within the keys [lo, hi], with the tokens above them
// holding `before` of the goal.
struct Ending {
  uint64_t lo, hi;
  double before, goal;
  bool all;     // nothing is cut
  int gathered; // the candidates hold every logit >= lo's: so many (0: they do not)
  __device__ __forceinline__ float edge() const { return key_logit(max_key(lo, (uint64_t)kMinKey << 32)); }
  __device__ __forceinline__ bool holds(uint64_t key) const { return key >= lo && key <= hi; }
};

// The prefix of the keys >= low0 that holds the tokens before which they hold
// less than goal tokens (!mass), or goal of their weight (mass): rounds until
// the keys it ends in are at most kList tokens.  After the first, if the whole
// prefix fits the candidates, rounds go over those.
template <typename T>
__device__ __forceinline__ Ending find_ending(const RowData<T>& row, const Scale& s, uint64_t low0, bool mass, double goal,
                                              Lds& lds) {
  const int lane = threadIdx.x & 63;
  Ending e = {low0, ((uint64_t)float_key(s.m) << 32) | 0xffffffffu, 0., goal, false, 0};
  const uint32_t tmin = (uint32_t)(low0 >> 32);
  const float least0 = key_float(max(tmin, kMinKey));
  // the first round goes from the top in steps of half an e-fold, the rest in the
  // last row; a later one divides its interval, or (open) goes on from its top in
  // steps of all the bins before
  float width = mass ? fminf(0.5f * s.temperature, kMaxFloat) : 0.5f;
  bool open = true;
  for (int round = 0;; ++round) {
    Bins b;
    b.n = e.gathered ? kFewBins : kBins;
    b.low = max((uint32_t)(e.lo >> 32), kMinKey);
    b.high = (uint32_t)(e.hi >> 32);
    b.low_index = max((uint32_t)e.lo, (uint32_t)~(row.vocab - 1));
    b.high_index = (uint32_t)e.hi;
    b.most = key_float(b.high);
    b.least = key_float(b.low);
    b.inv = 1.f / fmaxf(width, 1e-30f);
    b.top1 = __builtin_fmaf(b.most, b.inv, 1.f);
    b.by = b.low == b.high ? 2 : round < 4 && __builtin_isfinite(b.top1) ? 0 : 1;
    b.open = open && b.by == 0;
    const uint32_t range = b.by == 2 ? b.high_index - b.low_index : b.high - b.low;
    b.shift = 0;
    while ((range >> b.shift) >= (uint32_t)b.n) ++b.shift;

    __syncthreads();
    // The column is the thread's own: read, add, write.  (LDS additions without a
    // return take 176 cycles a wave here.)  Two logits at a time over the row, so
    // that two reads are on their way.
    // A list's order differs from run to run, so its weights are added as whole
    // numbers, of 2^-26 of the interval's largest (27 a thread at most), and what
    // is above the interval is known already.
    float* column = &lds.hist[0][threadIdx.x];
    uint32_t* few_column = &lds.few[0][threadIdx.x];
    int units = 0;  // a weight's, as a power of two
    if (e.gathered) {
      if (mass) units = min(26 - __builtin_amdgcn_frexp_expf(s.weight(b.most)), 126);
      for (int i = 0; i < b.n + 2; ++i) few_column[i * kThreads] = 0;
    } else {
      for (int i = 0; i < b.n + 2; ++i) column[i * kThreads] = 0.f;
    }
    const float unit = ldexpf(1.f, units);
    const auto put = [&](int i, float w) {
      if (!e.gathered) column[i * kThreads] += w;
      else if (i > 0) few_column[i * kThreads] += (uint32_t)(w * unit);
    };
    const auto put2 = [&](int i, float u, int j, float w) {
      const float a = column[i * kThreads], c = column[j * kThreads];
      column[i * kThreads] = a + u;
      column[j * kThreads] = (i == j ? a + u : c) + w;
    };
    const auto one_of = [&](float x) { return mass ? s.weight(x) : x > -INFINITY ? 1.f : 0.f; };
    const Source<T> from = {row, e.gathered ? lds.candidates : nullptr, e.gathered};
    if (round == 0 && b.by == 0 && tmin <= kMinKey) {
      row.each2([&](float x, float y) { put2(b.of_near(x), one_of(x), b.of_near(y), one_of(y)); });
    } else if (b.by == 0 && tmin <= kMinKey) {
      from.each([&](float x, int) { put(b.of_value(x), one_of(x)); });
    } else {
      from.each([&](float x, int i) {
        if (!(x >= least0)) return;
        const uint64_t key = order_key(x, i);
        if (key >= low0) put(b.of(key), mass ? s.weight(x) : 1.f);
      });
    }
    __syncthreads();
    // the rows' sums, a few a wave
    for (int q = threadIdx.x >> 6; q < b.n + 2; q += kWaves) {
      double t = 0.;
#pragma unroll
      for (int i = 0; i < kThreads / 64; ++i)
        t += e.gathered ? (double)lds.few[q][i * 64 + lane] : (double)lds.hist[q][i * 64 + lane];
#pragma unroll
      for (int o = 32; o; o >>= 1) t += __shfl_xor(t, o);
      if (lane == 0) lds.bins[q] = ldexp(t, -units);
    }
    __syncthreads();
    // every wave for itself, a lane a row: what the rows up to it hold
    const double mine = lane < b.n + 2 ? lds.bins[lane] : 0.;
    double upto = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double y = __shfl_up(upto, o);
      if (lane >= o) upto += y;
    }
    if (e.gathered) upto += e.before;
    if (round == 0) {
      const double total = __shfl(upto, 63);
      if (mass) e.goal *= total;
      e.all = !mass && total <= e.goal;
      if (e.all) return e;
    }
    // the row in which the goal is reached: one of the interval's that holds
    // anything, whatever the rounding of the sums says
    const uint64_t held_by = __ballot(lane >= 1 && lane <= (b.open ? b.n + 1 : b.n) && mine > 0.);
    if (held_by == 0) {
      e.all = true;
      return e;
    }
    const uint64_t reached = held_by & __ballot(upto >= e.goal);
    const int bin = reached ? __builtin_ctzll(reached) : 63 - __builtin_clzll(held_by);
    const double held = __shfl(mine, bin);
    e.before = __shfl(upto, bin) - held;
    // tokens of the prefix, at most: a row of the first round reaches down to e^(-i / 2)
    bool few = round == 0 && !mass && e.goal <= kCandidates;
    if (round == 0 && mass && b.open && bin <= b.n) {
      float tokens = lane <= bin ? (float)mine * exp2_fast(0.5f * kLog2e * lane) : 0.f;
#pragma unroll
      for (int o = 32; o; o >>= 1) tokens += __shfl_xor(tokens, o);
      few = 1.01f * tokens + 1.f <= kCandidates;
    }
    // the row's keys
    if (b.by == 2) {
      const uint32_t h = b.high_index - ((uint32_t)(bin - 1) << b.shift), span = (1u << b.shift) - 1;
      e.hi = ((uint64_t)b.high << 32) | h;
      e.lo = max_key(e.lo, ((uint64_t)b.high << 32) | (h > span ? h - span : 0u));
    } else {
      // where rows <= r begin, but for rounding
      const auto begin = [&](int r) {
        return b.by == 0 ? max(float_key(fmaxf(b.most - (float)r * (1.f / b.inv), -kMaxFloat)), kMinKey)
                         : b.high - min(b.high - b.low, (uint32_t)r << b.shift);
      };
      const uint32_t first = bin == b.n + 1 ? b.low
                                            : first_key(b.low, b.high, begin(bin), [&](uint32_t k) { return b.of_key(k) <= bin; });
      const uint32_t past = bin == 1 || b.of_key(b.high) >= bin
                                ? b.high
                                : first_key(b.low, b.high, begin(bin - 1), [&](uint32_t k) { return b.of_key(k) < bin; }) - 1;
      const uint64_t hi = ((uint64_t)past << 32) | 0xffffffffu;
      e.lo = max_key(e.lo, (uint64_t)first << 32);
      e.hi = hi < e.hi ? hi : e.hi;
    }
    if (few) {
      e.gathered = gather(row, e.edge(), lds);
      if (e.gathered > kCandidates) e.gathered = 0;
    }
    const float lightest = mass ? s.weight(e.edge()) : 1.f;
    if (held <= 0.99 * kList * (double)lightest) return e;
    open = b.open && bin == b.n + 1;
    width = open ? width * b.n : (key_logit(e.hi) - e.edge()) / (e.gathered ? kFewBins : kBins);
  }
}

// The keys of an ending into the list; returns how many (at most kList).
template <typename T>
__device__ __forceinline__ int list_ending(const RowData<T>& row, const Ending& e, Lds& lds) {
  __syncthreads();
  if (threadIdx.x == 0) lds.listed = 0;
  __syncthreads();
  const float least = e.edge(), most = key_logit(e.hi);
  const Source<T> from = {row, e.gathered ? lds.candidates : nullptr, e.gathered};
  from.each([&](float x, int i) {
    if (x >= least && x <= most) {
      const uint64_t key = order_key(x, i);
      if (e.holds(key)) {
        const int at = take_places(&lds.listed);
        if (at < kList) lds.list[at] = key;
      }
    }
  });
  __syncthreads();
  return min(lds.listed, kList);
}

// The prefix's last key, from the sorted list (n keys) of those it ends in.
__device__ __forceinline__ uint64_t last_key(const Scale& s, const Ending& e, bool mass, int n, Lds& lds) {
  sort_list(lds, n);
  const uint64_t mine = (int)threadIdx.x < n ? lds.list[threadIdx.x] : 0;
  const double part = mine == 0 ? 0. : mass ? (double)s.weight(key_logit(mine)) : 1.;
  double total;
  const double prior = e.before + block_scan(part, lds.wave_d, total);
  const uint64_t kept = mine != 0 && (prior < e.goal || threadIdx.x == 0) ? ~mine : 0;
  return ~block_reduce(kept, lds.wave_k, max_key);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_kernel(SampleParams p) {
  using L = Logits<T>;
  __shared__ Lds lds;
  const int r = blockIdx.x;
  RowData<T> row = {static_cast<const T*>(p.logits) + r * p.logits_stride, p.noise + r * p.noise_stride, p.vocab, false};
  const float temperature = p.temperature ? p.temperature[r] : p.temperature_all;
  int k = p.top_k ? p.top_k[r] : p.top_k_all;
  const float top_p = p.top_p ? p.top_p[r] : p.top_p_all;
  const float min_p = p.min_p ? p.min_p[r] : p.min_p_all;
  if (k >= p.vocab) k = 0;

  // The thread's maximum, the vectors where it first came up, and its sum of
  // 2^(l log2 e - its maximum's); a sum that is NaN tells of a logit that is, or
  // of +inf, and the pass is taken again.
  float mine, sum;
  int where;
  double total;
  Scale s;
  for (;;) {
    mine = -INFINITY;
    sum = 0.f;
    where = -1;
    row.batches([&](const u32x4 (&x)[4], int c) {
      float top = -INFINITY;
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int j = 0; j < L::N; ++j) top = fmaxf(top, L::get(x[u], j));
      if (top > mine) {
        sum *= mine == -INFINITY ? 0.f : exp2_fast((mine - top) * kLog2e);
        mine = top;
        where = c;
      }
      const float base = mine == -INFINITY ? 0.f : mine;
      float part = 0.f;
      if (fabsf(base) < 0x1p20f) {
        // l log2 e - base log2 e in one operation, and the rounding of the second
        // product, which is common to all, afterwards (up to 1/16 here; past 2^31 it
        // would leave the range of the exponential, and 0 times infinity)
        const float product = base * kLog2e;
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int j = 0; j < L::N; ++j) part += exp2_fast(__builtin_fmaf(L::get(x[u], j), kLog2e, -product));
        part *= exp2_fast(-__builtin_fmaf(base, kLog2e, -product));
      } else {
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int j = 0; j < L::N; ++j) part += exp2_fast((L::get(x[u], j) - base) * kLog2e);
      }
      sum += part;
    });
    if (row.rest() >= 0) {
      const float x = row.one(row.rest());
      const float top = fmaxf(mine, x), base = top == -INFINITY ? 0.f : top;
      sum = (mine == -INFINITY ? 0.f : sum * exp2_fast((mine - base) * kLog2e)) + exp2_fast((x - base) * kLog2e);
      if (top > mine) where = p.vocab;
      mine = top;
    }
    const float m = block_reduce(mine, lds.wave_f, max_float);
    total = block_reduce(mine == -INFINITY && sum == 0.f ? 0. : (double)(sum * exp2_fast((mine - m) * kLog2e)), lds.wave_d,
                         add_double);
    if (row.odd || total < INFINITY) {  // (a row of -inf alone has the sum 0)
      s.init(m, temperature);
      break;
    }
    row.odd = true;
  }
  if (!(s.m > -INFINITY)) {
    if (threadIdx.x == 0) {
      p.token[r] = -1;
      p.logprob[r] = -INFINITY;
    }
    return;
  }

  uint64_t pick = 0;  // the best score's key, then its token's index complemented
  const auto take = [&](float z, float g, int i) {
    const float t = z + g;
    if (t > -INFINITY) pick = max_key(pick, ((uint64_t)float_key(fminf(t, kMaxFloat)) << 32) | (uint32_t)~i);
  };
  const auto score = [&](uint64_t key, float g) {
    const float z = s.z(key_logit(key));
    if (min_p <= 0.f || expf(z) >= min_p) take(z, g, key_index(key));
  };
  // the candidates that a prefix ending with low keeps
  const auto score_candidates = [&](int n, uint64_t low) {
    constexpr int U = 4;
    for (int i = threadIdx.x; i < n; i += U * kThreads) {
      int at[U];
      float x[U], g[U];
#pragma unroll
      for (int u = 0; u < U; ++u) at[u] = (int)lds.candidates[i + u * kThreads < n ? i + u * kThreads : i];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        x[u] = row.one(at[u]);
        g[u] = row.noise[at[u]];
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {  // (one twice: no harm)
        const uint64_t key = order_key(x[u], at[u]);
        if (key >= low) score(key, g[u]);
      }
    }
  };

  if (temperature > 0.f) {
    bool done = false;
    if (k > 0 && k <= kList) {
      const float least = key_float(max((k <= kRanked ? reached_by_waves(float_key(mine) >> 16, k, lds)
                                                       : reached_by(float_key(mine) >> 16, k, lds)) << 16, kMinKey));
      const int n = gather(row, least, lds);
      if (n <= kList) {
        if ((int)threadIdx.x < n) {
          const int i = lds.candidates[threadIdx.x];
          lds.list[threadIdx.x] = order_key(row.one(i), i);
        }
        sort_list(lds, n);
        const uint64_t key = (int)threadIdx.x < min(n, k) ? lds.list[threadIdx.x] : 0;
        bool keep = key != 0;
        if (top_p < 1.f) {
          double held;
          const double before = block_scan(keep ? (double)s.weight(key_logit(key)) : 0., lds.wave_d, held);
          keep = keep && (before < (double)top_p * held || threadIdx.x == 0);
        }
        if (keep) score(key, row.noise[key_index(key)]);
        done = true;
      }
    }
    if (!done) {
      // what a logit must reach for min_p, but for rounding
      float least = -kMaxFloat;
      if (min_p > 0.f) {
        const float d = temperature * logf(min_p);
        least = fmaxf(least, s.m + d - 1e-5f * (fabsf(s.m) + fabsf(d) + temperature));
      }
      uint64_t low = 1;  // the prefix's last key
      int gathered = 0;
      if (k > 0) {
        const Ending e = find_ending(row, s, low, false, (double)k, lds);
        if (!e.all) low = last_key(s, e, false, list_ending(row, e, lds), lds);
      }
      if (top_p < 1.f) {
        const Ending e = find_ending(row, s, low, true, (double)top_p, lds);
        if (!e.all) low = last_key(s, e, true, list_ending(row, e, lds), lds);
        gathered = e.all ? 0 : e.gathered;
      }
      least = fmaxf(least, key_float(max((uint32_t)(low >> 32), kMinKey)));
      if (!gathered && ((k > 0 && k <= kCandidates) || (min_p > 0.f && top_p >= 1.f))) {  // it may fit
        gathered = gather(row, least, lds);
        if (gathered > kCandidates) gathered = 0;
      }
      if (gathered) {
        score_candidates(gathered, low);
      } else {
        // too many for a list: every logit's score.  A thread's indices rise, so the
        // first of equal scores stays; what beats the best so far is rare, and only
        // that is looked at closely.
        float best = -INFINITY;
        int at = 0;
        const uint32_t edge = (uint32_t)(low >> 32);
        const auto dense = [&](float x, float z, float g, int i) {
          const float t = z + g;
          if (t > best && x >= least)
            if (float_key(x) > edge || order_key(x, i) >= low)
              if (min_p <= 0.f || expf(s.z(x)) >= min_p) {
                best = t;
                at = i;
              }
        };
        if (s.inv != 0.f) row.each_with_noise([&](float x, float g, int i) { dense(x, s.z_fast(x), g, i); });
        else row.each_with_noise([&](float x, float g, int i) { dense(x, s.z(x), g, i); });
        if (best > -INFINITY) pick = ((uint64_t)float_key(fminf(best, kMaxFloat)) << 32) | (uint32_t)~at;
      }
    }
    pick = block_reduce(pick, lds.wave_k, max_key);
  }
  if (pick == 0) {  // the first of the order: greedy, or noise that nothing wins
    if (mine == s.m) {
      if (where == p.vocab) {
        pick = (1ull << 32) | (uint32_t)~(row.vectors() * L::N + (int)threadIdx.x);
      } else {
        u32x4 x[4];
        row.load(x, where);
#pragma unroll
        for (int u = 3; u >= 0; --u)
#pragma unroll
          for (int j = L::N - 1; j >= 0; --j)
            if (L::get(x[u], j) == s.m) pick = (1ull << 32) | (uint32_t)~((where + u * kThreads) * L::N + j);
      }
    }
    pick = block_reduce(pick, lds.wave_k, max_key);
  }
  if (threadIdx.x == 0) {
    const int token = key_index(pick);
    p.token[r] = token;
    p.logprob[r] = (row.one(token) - s.m) - (float)log(total);
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
