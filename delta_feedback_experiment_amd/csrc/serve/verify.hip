// Verification of drafted tokens against the target's probabilities, from given
// random numbers (gfx950).
//
// p = softmax(l / T) in the row after a draft's place, q the same of the draft's
// own logits (or 1 at the draft).  Drafts are accepted in turn while u q(d) < p(d);
// the next token maximises log max(p - q, 0) + noise in the first row whose draft
// is not, log p + noise in the last row and in one without a draft, where nothing was
// drawn from q (the Gumbel numbers make that a draw).
//
// Bound by the logits' bytes.  Two launches.  The first reads every row of the
// target and of the drafts once, a row over several workgroups, and leaves each
// piece's maximum m and sum of 2^((l - m) c), c = log2 e / T: whether a row is
// reached is known only after those before it, and reading it anyway costs less
// than a trip to memory per draft.  In the second, every workgroup of a sequence
// joins the pieces of its rows, eight rows at a time, until a draft is not accepted,
// and scans its part of that one row; the parts' best, the lowest index of the
// highest score, does not depend on their order.
//
// Sums are FP32: a thread's, the wave's in pairs, the pieces' in pairs.
//
// Measured, BF16: 64 sequences of up to 5 drafts, 131,072 tokens, 322 rows and 258 of
// the drafts': 33 us for the sums (152 MB, 4.6 TB/s) and 21 for the picks (50 MB, behind
// three trips to memory one after another).
#include "logits.h"
#include "paged_common.h"

namespace pkda {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kMaxPieces = 64;  // of a row: one a lane where they are joined
constexpr int kVectors = 2;     // of 16 bytes a thread asks for at a time
constexpr int kMaxVocab = 1 << 24;

struct Sum {  // a piece of a row
  float m, s;      // maximum and sum of the target's
  float dm, ds;    // and of the draft's
  int first;       // lowest index of the target's maximum
  int drafted;     // in a row's first piece: the row's draft, -1 for none that can be taken,
  float l, dl;     // and its logits
};
// A score and its token as one number, so that the larger is the better: the
// score's order, then the lower index.  0: none.
struct Best {
  uint64_t key;
  __device__ __forceinline__ static uint64_t of(float score, int index) {
    const uint32_t b = __float_as_uint(score + 0.f);
    return (uint64_t)(b & 0x80000000u ? ~b : b | 0x80000000u) << 32 | (uint32_t)~index;
  }
  __device__ __forceinline__ int index() const { return (int)~(uint32_t)key; }
};

struct VerifyParams {
  const void *logits, *draft;
  int64_t logits_stride, draft_stride, noise_stride;
  const int32_t* drafts;
  const float *uniform, *noise, *temperature;
  float temperature_all;
  const int32_t* cu;
  int rows, vocab, num_seqs;
  int pieces;  // of a row, in the first kernel
  int parts;   // of the last row, in the second
  int32_t *tokens, *accepted;
  Sum* sums;   // [rows][pieces]
  uint64_t* best;  // [num_seqs] of the parts that are done
  int32_t* done;   // [num_seqs] how many those are
};

// One logit as the rows' vectors are taken: +inf is the largest number of its own type.
template <typename T>
__device__ __forceinline__ float one_logit(const T* l, int i) {
  return fminf(usable(io<T>::load(l + i)), __uint_as_float(sizeof(T) == 2 ? 0x7f7f0000u : 0x7f7fffffu));
}

__device__ __forceinline__ int row_bound(const VerifyParams& p, int n) {
  return n == 0 ? 0 : clamp_int(p.cu[n], 0, p.rows);
}
__device__ __forceinline__ float temperature_of(const VerifyParams& p, int n) {
  return p.temperature ? p.temperature[n] : p.temperature_all;
}
// c = log2 e / T, a number for the smallest T too.
__device__ __forceinline__ float exponent_factor(float t) { return fminf(kLog2e / t, kMaxFloat); }

// Vector v of a row of `vocab` logits; what is past the row is -inf.
template <typename T>
__device__ __forceinline__ u32x4 row_vector(const T* l, int v, int vocab) {
  using L = Logits<T>;
  if ((v + 1) * L::N <= vocab) return reinterpret_cast<const u32x4_any*>(l)[v];
  u32x4 x = {L::none, L::none, L::none, L::none};
  for (int j = 0; j < L::N; ++j) {
    const int i = v * L::N + j;
    if (i >= vocab) break;
    if constexpr (sizeof(T) == 2) x[j / 2] = j & 1 ? (x[j / 2] & 0xffffu) | ((uint32_t)l[i] << 16) : (x[j / 2] & 0xffff0000u) | l[i];
    else x[j] = __float_as_uint(l[i]);
  }
  return x;
}

// (m, s) of two sets of numbers joined.
__device__ __forceinline__ float carried(float m, float to, float c) {
  return m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(fmaxf(m - to, -kMaxFloat) * c);
}
__device__ __forceinline__ void join_sum(float& m, float& s, float m1, float s1, float c) {
  const float to = fmaxf(m, m1);
  s = s * carried(m, to, c) + s1 * carried(m1, to, c);
  m = to;
}

// A thread's maximum and sum over its vectors.  First as if all were numbers; a
// NaN or +inf among them, or nothing at all, shows in the sum.
template <typename T, int U>
__device__ __forceinline__ void vectors_sum(u32x4 (&x)[U], float c, float& m, float& s) {
  using L = Logits<T>;
  m = -INFINITY;
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int j = 0; j < L::N; ++j) m = fmaxf(m, L::get(x[u], j));
  s = 0.f;
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int j = 0; j < L::N; ++j) s += __builtin_amdgcn_exp2f((L::get(x[u], j) - m) * c);
  if (!(s < INFINITY)) {
    m = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      L::clean(x[u]);
#pragma unroll
      for (int j = 0; j < L::N; ++j) m = fmaxf(m, L::get(x[u], j));
    }
    s = 0.f;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < L::N; ++j) s += carried(L::get(x[u], j), m, c);
  }
}

// The workgroup's threads' (m, s) joined; every thread gets it.
__device__ __forceinline__ void block_sum(float& m, float& s, float c, float (&lds)[2 * kWaves]) {
#pragma unroll
  for (int o = 32; o; o >>= 1) join_sum(m, s, __shfl_xor(m, o), __shfl_xor(s, o), c);
  const int w = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) {
    lds[2 * w] = m;
    lds[2 * w + 1] = s;
  }
  __syncthreads();
  m = lds[0];
  s = lds[1];
#pragma unroll
  for (int i = 1; i < kWaves; ++i) join_sum(m, s, lds[2 * i], lds[2 * i + 1], c);
}

// ---------------------------------------------------------------------------
// Every row's pieces.
// ---------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(kThreads) void verify_sums_kernel(VerifyParams p) {
  using L = Logits<T>;
  constexpr int U = kVectors;
  __shared__ float s_sum[2][2 * kWaves];
  __shared__ int s_first[kWaves];
  const int piece = blockIdx.x % p.pieces, row = blockIdx.x / p.pieces, tid = threadIdx.x;
  if (piece == 0)
    for (int64_t i = (int64_t)row * kThreads + tid; i < p.num_seqs; i += (int64_t)p.rows * kThreads) {
      p.best[i] = 0;
      p.done[i] = 0;
    }
  const int n = wave_upper(p.num_seqs, row, [&](int i) -> int64_t { return row_bound(p, i); });
  if (n >= p.num_seqs) {  // a row of no sequence
    if (piece == 0 && tid == 0) p.tokens[row] = -1;
    return;
  }
  const float t = temperature_of(p, n), c = exponent_factor(t);
  const bool greedy = t <= 0.f;
  const T* l = static_cast<const T*>(p.logits) + row * p.logits_stride;
  // the last row's draft, and a greedy row's draft logits, are not asked for
  const T* d = p.draft && !greedy && row + 1 < row_bound(p, n + 1) ? static_cast<const T*>(p.draft) + row * p.draft_stride : nullptr;
  const int vectors = (p.vocab + L::N - 1) / L::N, chunks = (vectors + kThreads * U - 1) / (kThreads * U);
  // the draft's own logits, while the row's are on their way
  Sum r;
  r.drafted = -1;
  r.l = r.dl = -INFINITY;
  if (piece == 0 && tid == 0) {
    const int i = p.drafts[row];
    if ((unsigned)i < (unsigned)p.vocab) {
      r.drafted = i;
      r.l = one_logit(l, i);
      if (d) r.dl = one_logit(d, i);
    }
  }
  float m = -INFINITY, s = 0.f, dm = -INFINITY, ds = 0.f;
  int first = INT32_MAX;
  for (int k = piece; k < chunks; k += p.pieces) {
    const int v0 = k * kThreads * U + tid;
    u32x4 x[U], y[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      x[u] = y[u] = u32x4{L::none, L::none, L::none, L::none};
      const int v = v0 + u * kThreads;
      if (v < vectors) {
        x[u] = row_vector<T>(l, v, p.vocab);
        if (d) y[u] = row_vector<T>(d, v, p.vocab);
      }
    }
    if (greedy) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        L::clean(x[u]);
#pragma unroll
        for (int j = 0; j < L::N; ++j) {
          const float a = L::get(x[u], j);
          if (a > m) {
            m = a;
            first = (v0 + u * kThreads) * L::N + j;
          }
        }
      }
      continue;
    }
    float m1, s1;
    vectors_sum<T, U>(x, c, m1, s1);
    join_sum(m, s, m1, s1, c);
    if (d) {
      vectors_sum<T, U>(y, c, m1, s1);
      join_sum(dm, ds, m1, s1, c);
    }
  }
  if (greedy) {
    float top = m;
#pragma unroll
    for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    if (m != top || top == -INFINITY) first = INT32_MAX;
#pragma unroll
    for (int o = 32; o; o >>= 1) first = min(first, __shfl_xor(first, o));
    if ((tid & 63) == 0) {
      s_sum[0][tid >> 6] = top;
      s_first[tid >> 6] = first;
    }
    __syncthreads();
    m = s_sum[0][0];
    for (int i = 1; i < kWaves; ++i) m = fmaxf(m, s_sum[0][i]);
    first = INT32_MAX;
    for (int i = 0; i < kWaves; ++i)
      if (s_sum[0][i] == m) first = min(first, s_first[i]);
  } else {
    block_sum(m, s, c, s_sum[0]);
    if (d) block_sum(dm, ds, c, s_sum[1]);
  }
  if (tid == 0) {
    r.m = m; r.s = s; r.dm = dm; r.ds = ds; r.first = first;
    p.sums[(int64_t)row * p.pieces + piece] = r;
  }
}

// ---------------------------------------------------------------------------
// The drafts in turn, and the next token.
// ---------------------------------------------------------------------------
struct RowSum {
  float m, s, dm, ds;
  int first;
  int drafted;  // lane 0's: the row's draft, -1 for none that can be taken
};
// f over the wave's x, every lane getting it.
template <typename V, typename F>
__device__ __forceinline__ V wave_all(V x, F f) {
  const auto moved = [&](auto move) { return __builtin_bit_cast(V, move(__builtin_bit_cast(int, x))); };
  x = f(x, moved([](int i) { return __builtin_amdgcn_update_dpp(0, i, 0xB1, 0xF, 0xF, false); }));   // quad [1,0,3,2]
  x = f(x, moved([](int i) { return __builtin_amdgcn_update_dpp(0, i, 0x4E, 0xF, 0xF, false); }));   // quad [2,3,0,1]
  x = f(x, moved([](int i) { return __builtin_amdgcn_update_dpp(0, i, 0x141, 0xF, 0xF, false); }));  // half-row mirror
  x = f(x, moved([](int i) { return __builtin_amdgcn_update_dpp(0, i, 0x140, 0xF, 0xF, false); }));  // row mirror
  int i = __builtin_bit_cast(int, x);
  auto r = __builtin_amdgcn_permlane16_swap(i, i, false, false);
  x = f(__builtin_bit_cast(V, (int)r[0]), __builtin_bit_cast(V, (int)r[1]));
  i = __builtin_bit_cast(int, x);
  r = __builtin_amdgcn_permlane32_swap(i, i, false, false);
  return f(__builtin_bit_cast(V, (int)r[0]), __builtin_bit_cast(V, (int)r[1]));
}
__device__ __forceinline__ float wave_max(float x) {
  return wave_all(x, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float wave_total(float x) {
  return wave_all(x, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ int wave_min(int x) {
  return wave_all(x, [](int a, int b) { return min(a, b); });
}
// A row's piece of this lane.
__device__ __forceinline__ Sum lane_piece(const VerifyParams& p, int row) {
  const int lane = threadIdx.x & 63;
  Sum x;
  x.m = x.dm = x.l = x.dl = -INFINITY;
  x.s = x.ds = 0.f;
  x.first = INT32_MAX;
  x.drafted = -1;
  if (lane < p.pieces) x = p.sums[(int64_t)row * p.pieces + lane];
  return x;
}
// A row's pieces joined, by a wave.
__device__ __forceinline__ RowSum row_sum(const Sum& x, float c) {
  RowSum r;
  r.m = wave_max(x.m);
  r.dm = wave_max(x.dm);
  r.s = wave_total(x.s * carried(x.m, r.m, c));
  r.ds = wave_total(x.ds * carried(x.dm, r.dm, c));
  r.first = wave_min(x.m == r.m ? x.first : INT32_MAX);
  r.drafted = x.drafted;
  return r;
}
__device__ __forceinline__ Best block_best(Best b, Best (&lds)[kWaves]) {
#pragma unroll
  for (int o = 32; o; o >>= 1) {
    const uint64_t other = __shfl_xor((unsigned long long)b.key, o);
    b.key = max(b.key, other);
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = b;
  __syncthreads();
  b = lds[0];
#pragma unroll
  for (int i = 1; i < kWaves; ++i) b.key = max(b.key, lds[i].key);
  return b;
}

// a b - q with the product rounded, as q is: where p and q are the same number
// nothing is left.
__device__ __forceinline__ float difference(float a, float b, float q) {
#pragma clang fp contract(off)
  const float p = a * b;
  return p - q;
}

// ln x for x > 0 on the hardware log2, which takes no denormal numbers.
__device__ __forceinline__ float log_of(float x) {
  const bool small = x < 0x1p-96f;
  const float l = __builtin_amdgcn_logf(small ? x * 0x1p64f : x);
  return (small ? l - 64.f : l) * 0.693147180559945309f;
}

// The scores of a row's vectors part, part + parts, ... (in workgroups).  left: of
// what p has more than q; otherwise of p but for `without`.
template <typename T>
__device__ __forceinline__ Best scan_row(const VerifyParams& p, const T* l, const T* d, const float* noise, float t,
                                         const RowSum& r, bool left, int without, int part, int parts) {
  using L = Logits<T>;
  const int vectors = (p.vocab + L::N - 1) / L::N;
  const float inv_t = fminf(1.f / t, kMaxFloat), c = exponent_factor(t);
  const float ps = 1.f / r.s, qs = r.ds > 0.f ? 1.f / r.ds : 0.f;
  // x / T, the product's rounding made good where T is no power of two
  const auto over_t = [&](float x) {
    const float y = x * inv_t, e = __builtin_fmaf(-y, t, x);
    return fabsf(e) < INFINITY ? __builtin_fmaf(e, inv_t, y) : y;
  };
  float best = 0.f;
  int index = -1;
  constexpr int U = kVectors, NV = L::N / 4;
  for (int v0 = part * kThreads + threadIdx.x; v0 < vectors; v0 += U * parts * kThreads) {
    u32x4 x[U], y[U], g[U][NV];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int v = v0 + u * parts * kThreads;
      x[u] = y[u] = u32x4{L::none, L::none, L::none, L::none};
      if (v >= vectors) continue;
      x[u] = row_vector<T>(l, v, p.vocab);
      if (left) y[u] = row_vector<T>(d, v, p.vocab);
#pragma unroll
      for (int j = 0; j < NV; ++j) g[u][j] = row_vector<float>(noise, v * NV + j, p.vocab);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int j = 0; j < L::N; ++j) {
        const int i = (v0 + u * parts * kThreads) * L::N + j;
        const float lx = L::get(x[u], j);
        bool in = lx > -INFINITY && i != without;
        const float above = fmaxf(fminf(lx, r.m) - r.m, -kMaxFloat);  // (+inf is the row's maximum)
        float score;
        if (left) {
          const float ly = L::get(y[u], j);
          const float q = ly > -INFINITY ? __builtin_amdgcn_exp2f(fmaxf(fminf(ly, r.dm) - r.dm, -kMaxFloat) * c) * qs : 0.f;
          const float rest = difference(__builtin_amdgcn_exp2f(above * c), ps, q);
          in = in && rest > 0.f;
          score = log_of(rest);
        } else {
          score = over_t(above);
        }
        score += __uint_as_float(g[u][j / 4][j % 4]);
        if (in && (score > best || (index < 0 && score == score))) {  // (a thread's indices rise)
          best = score;
          index = i;
        }
      }
    }
  }
  return {index < 0 ? 0 : Best::of(best, index)};
}

template <typename T>
__global__ __launch_bounds__(kThreads) void verify_pick_kernel(VerifyParams p) {
  constexpr int kRows = 2;  // of a wave at a time
  __shared__ RowSum s_row[kRows * kWaves];
  __shared__ int s_stop[kRows * kWaves];
  __shared__ Best s_best[kWaves];
  __shared__ int s_last;
  const int part = blockIdx.x % p.parts, n = blockIdx.x / p.parts, tid = threadIdx.x;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int first = row_bound(p, n), count = max(0, row_bound(p, n + 1) - first);
  if (count == 0) {
    if (part == 0 && tid == 0) p.accepted[n] = 0;
    return;
  }
  const float t = temperature_of(p, n), c = exponent_factor(t);
  const bool greedy = t <= 0.f;
  const T* logits = static_cast<const T*>(p.logits);
  const T* draft = static_cast<const T*>(p.draft);
  RowSum r;
  int stop = count - 1;
  for (int j0 = 0; j0 < count; j0 += kRows * kWaves) {
    // everything of a wave's rows is asked for before any of it is waited for
    Sum x[kRows];
    float u[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int row = first + min(j0 + i * kWaves + w, count - 1);
      u[i] = p.uniform[row];
      x[i] = lane_piece(p, row);
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int j = j0 + i * kWaves + w;
      const RowSum y = row_sum(x[i], c);
      if ((tid & 63) == 0) {  // whose piece is the row's first
        const Sum& z = x[i];
        bool taken = false;
        if (j + 1 < count && z.drafted >= 0) {
          if (greedy) {
            taken = z.drafted == y.first;
          } else {
            const float pd = z.l > -INFINITY && y.s > 0.f ? carried(z.l, y.m, c) / y.s : 0.f;
            const float qd = !draft ? 1.f : z.dl > -INFINITY && y.ds > 0.f ? carried(z.dl, y.dm, c) / y.ds : 0.f;
            taken = u[i] * qd < pd;
          }
        }
        s_row[i * kWaves + w] = y;
        s_stop[i * kWaves + w] = j < count && !taken;
      }
    }
    __syncthreads();
    int at = -1;
#pragma unroll
    for (int i = kRows * kWaves - 1; i >= 0; --i)
      if (s_stop[i]) at = i;
    if (at >= 0) {
      r = s_row[at];
      stop = j0 + at;
      break;
    }
    __syncthreads();
  }
  const int row = first + stop;
  int token = -1;
  bool last = part == 0;  // whether this workgroup writes the result
  if (greedy) {
    token = r.first == INT32_MAX ? -1 : r.first;
  } else if (r.s > 0.f) {
    const T* l = logits + row * p.logits_stride;
    const T* q = draft ? draft + row * p.draft_stride : nullptr;
    const float* noise = p.noise + n * p.noise_stride;
    const bool rejected = stop + 1 < count;
    const bool left = rejected && q && r.drafted >= 0;  // (else nothing was drawn from q)
    const int without = rejected && !q ? r.drafted : -1;
    Best b = block_best(scan_row<T>(p, l, q, noise, t, r, left, without, part, p.parts), s_best);
    if (p.parts > 1) {
      // The parts' best by one atomic maximum: nothing but atomics passes between
      // the workgroups, so that none has to write its cache back, and the count
      // goes out when the maximum has come back.
      if (tid == 0) {
        __hip_atomic_fetch_max(p.best + n, b.key, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        s_last = __hip_atomic_fetch_add(p.done + n, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == p.parts - 1;
      }
      __syncthreads();
      last = s_last;
      if (!last) return;
      b.key = __hip_atomic_load(p.best + n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    // nothing of p is left: p itself, by this workgroup alone
    if (b.key == 0 && rejected) b = block_best(scan_row<T>(p, l, q, noise, t, r, false, -1, 0, 1), s_best);
    token = b.key == 0 ? -1 : b.index();
  }
  if (!last) return;
  for (int j = tid; j < count; j += kThreads) p.tokens[first + j] = j < stop ? p.drafts[first + j] : j == stop ? token : -1;
  if (tid == 0) p.accepted[n] = stop;
}

// Pieces of a row, and parts of a sequence's last one: enough workgroups for the
// card, none with less than a vector a thread.
void verify_plan(VerifyParams& p, int dtype) {
  const int64_t n = dtype == PKDA_BF16 ? 8 : 4, vectors = (p.vocab + n - 1) / n;
  const auto pieces = [&](int64_t rows, int64_t each, int64_t blocks) {
    int64_t want = (blocks + rows - 1) / (rows > 0 ? rows : 1);
    const int64_t cap = (vectors + each - 1) / each;
    want = want < cap ? want : cap;
    return (int)(want < 1 ? 1 : want < kMaxPieces ? want : kMaxPieces);
  };
  // A part's way to its row is some trips to memory, however little it then scans:
  // 64 sequences of 131,072 tokens, 64 parts each 59 us, 16 parts 55, 8 parts 60 (in
  // all); 32 of 50,304 31, 27 and 25 with 50, 32 and 16.
  p.pieces = pieces(p.rows, kThreads * kVectors, 4096);
  p.parts = pieces(p.num_seqs, kThreads, 768);
}
int64_t verify_floats(const VerifyParams& p) {
  return (int64_t)p.rows * p.pieces * (int64_t)(sizeof(Sum) / 4) + (int64_t)p.num_seqs * 3;
}
int verify_sizes(const pkda_verify_args* a, VerifyParams& p) {
  PKDA_REQUIRE(a != nullptr, PKDA_EINVAL, "null args");
  PKDA_REQUIRE(a->struct_size == (int32_t)sizeof(*a), PKDA_EINVAL, "pkda_verify_args size mismatch");
  PKDA_REQUIRE(a->dtype == PKDA_F32 || a->dtype == PKDA_BF16, PKDA_EUNSUPPORTED, "dtype %d", a->dtype);
  PKDA_REQUIRE(a->rows >= 0 && a->num_seqs >= 0, PKDA_EINVAL, "rows %d, num_seqs %d", a->rows, a->num_seqs);
  PKDA_REQUIRE(a->vocab >= 1 && a->vocab <= kMaxVocab, PKDA_EINVAL, "vocab %d (1 .. 2^24)", a->vocab);
  p.rows = a->rows; p.vocab = a->vocab; p.num_seqs = a->num_seqs;
  verify_plan(p, a->dtype);
  PKDA_REQUIRE((int64_t)p.rows * p.pieces <= INT32_MAX && (int64_t)p.num_seqs * p.parts <= INT32_MAX, PKDA_EINVAL,
               "%d rows of %d sequences", p.rows, p.num_seqs);
  return 0;
}

}  // namespace
}  // namespace pkda

extern "C" int64_t pkda_verify_workspace(const pkda_verify_args* a) {
  pkda::VerifyParams p;
  if (pkda::verify_sizes(a, p)) return -1;
  return pkda::verify_floats(p);
}

extern "C" int pkda_verify(const pkda_verify_args* a, void* stream) {
  using namespace pkda;
  VerifyParams p;
  if (int st = verify_sizes(a, p)) return st;
  PKDA_REQUIRE(a->cu_seqlens, PKDA_EINVAL, "null cu_seqlens");
  if (a->rows == 0 && a->num_seqs == 0) return 0;
  PKDA_REQUIRE(a->num_seqs == 0 || (a->accepted && a->noise), PKDA_EINVAL, "null tensor");
  PKDA_REQUIRE(a->rows == 0 || (a->logits && a->drafts && a->uniform && a->tokens), PKDA_EINVAL, "null tensor");
  PKDA_REQUIRE(a->workspace && (uintptr_t)a->workspace % 16 == 0, PKDA_EINVAL, "workspace");
  const int64_t size = a->dtype == PKDA_BF16 ? 2 : 4;
  PKDA_REQUIRE(((uintptr_t)a->logits | (uintptr_t)a->draft_logits) % size == 0 && (uintptr_t)a->noise % 4 == 0, PKDA_EINVAL,
               "logits and noise must be aligned to their numbers");
  p.logits = a->logits; p.logits_stride = a->logits_stride;
  p.draft = a->draft_logits; p.draft_stride = a->draft_stride;
  p.drafts = a->drafts; p.uniform = a->uniform; p.noise = a->noise; p.noise_stride = a->noise_stride;
  p.cu = a->cu_seqlens; p.temperature = a->temperature; p.temperature_all = a->temperature_all;
  p.tokens = a->tokens; p.accepted = a->accepted;
  p.sums = reinterpret_cast<Sum*>(a->workspace);
  p.best = reinterpret_cast<uint64_t*>(p.sums + (int64_t)p.rows * p.pieces);
  p.done = reinterpret_cast<int32_t*>(p.best + p.num_seqs);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 block(kThreads);
  if (p.rows > 0) {
    const dim3 grid((unsigned)(p.rows * p.pieces));
    if (a->dtype == PKDA_BF16) hipLaunchKernelGGL(verify_sums_kernel<bf16_t>, grid, block, 0, s, p);
    else hipLaunchKernelGGL(verify_sums_kernel<float>, grid, block, 0, s, p);
    if (int st = launch_status("pkda_verify")) return st;
  }
  if (p.num_seqs == 0) return 0;
  const dim3 grid((unsigned)(p.num_seqs * p.parts));
  if (a->dtype == PKDA_BF16) hipLaunchKernelGGL(verify_pick_kernel<bf16_t>, grid, block, 0, s, p);
  else hipLaunchKernelGGL(verify_pick_kernel<float>, grid, block, 0, s, p);
  return launch_status("pkda_verify(pick)");
}
