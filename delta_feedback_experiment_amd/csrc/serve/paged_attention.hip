// Attention of new tokens over a paged key/value cache (gfx950).
//
// Rows.  The group = q_heads / kv_heads query heads of one key/value head share
// its keys, so a workgroup's tile is rows of (token, query head of the group)
// of one sequence, tokens slowest: a single token fills group rows, a chunk
// any number.  Scores, softmax and output run in one pass over the keys with
// the row's running maximum m and sum l (base 2, FP32):
//   m' = max(m, max_s S),  p = 2^(S - m'),  l = l 2^(m - m') + sum_s p,
//   O = O 2^(m - m') + p V,   o = O / l,  lse = (m + log2 l) ln 2.
//
// Products.  Both are taken transposed, S^T = K Q^T and O^T = V^T P^T, as
// 32x32 MFMA tiles.  A lane then holds one query row (its column) and 16 of a
// tile's 32 keys, so a row's maximum and sum are a lane's own and one exchange
// between the wave's halves, the rescaling of O is a multiply by the lane's own
// factor, and P^T is already the second product's operand: the accumulator's
// key order, 8 (r / 4) + 4 half + r % 4 for register r, is the order in which
// the product reads V's rows.  K, Q and V keep their 16-byte chunks: chunk 2 i +
// half of a row is operand i of the lane's half (BF16: one 32x32x16 step; FP32:
// four 32x32x2 steps).
//
// Two forms, in one launch.  Up to 32 rows of a sequence (decode, a few proposed
// tokens): four waves take 32 keys each in turn, each with its own m, l and O,
// and join at the end; keys go straight from memory to operand registers, values
// through a wave's own piece of LDS (the transposing reads), the next tile's
// loads in flight during a tile's arithmetic.  More rows (a chunk): four waves of
// 32 rows share tiles of 64 keys staged in LDS, double-buffered.  Where rows are
// few, a sequence's keys are split over workgroups and a second kernel joins the
// parts.
//
// Roundings to BF16: the probabilities, as the second product's operand (their
// sum l is of the unrounded ones), and the output; scores, m, l and O are FP32.
//
// What bounds it, measured in BF16 with heads of 128 (a large read runs at 4.0 to
// 5.0 TB/s, a large matrix product at 1188 TFLOP/s).  Decode, 256 sequences of
// 2,600 keys, 32/8 heads: 546 us, 4.98 TB/s of keys and values.  One sequence of
// 131,072 keys: 114 us, 4.7 TB/s.  2,048 tokens after 14,336, 32/8 heads: 603 us,
// 855 TFLOP/s: a wave's 32 products a tile are 1,024 cycles, its 246 vector
// instructions, 32 exponentials among them, about 1,370, and its reads of LDS
// about 800; the other workgroup's wave on the SIMD overlaps them only in part
// (2,500 cycles a tile and wave).  13 prompts of 250 to 1,659 tokens, 16/4 heads:
// 87 us, 588 TFLOP/s: 6 us of a row tile's 33 are its way to its first keys and
// its output.
#include <math.h>

#include "paged_common.h"

namespace pkda {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kMaxSplits = 256;
constexpr int kMinChunk = 128;  // a split is a multiple of so many keys

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) bf16x4 lds_bf16x4;

struct AttnParams {
  PagedSeqs s;
  const void* q;
  int64_t q_stride;
  const void *k_pages, *v_pages;
  int64_t k_page_stride, v_page_stride;
  int q_heads, kv_heads;
  FastDiv group;
  float scale2;  // |scale| log2 e: the softmax is taken in base 2
  bool negate;   // scale < 0: queries are negated
  int splits;
  int min_chunk;       // keys of a split, at least
  int whole;           // sequences of up to so many positions are not split
  int key_rows;        // sequences of up to so many rows run with their keys over the waves
  unsigned row_blocks; // workgroups of the others, before those
  void* o;
  float* lse;
  float* part_o;   // [splits][num_tokens * q_heads][head_dim]
  float* part_ml;  // [splits][num_tokens * q_heads][2]
};

template <typename T, int D> struct Geo {
  static constexpr int RB = D * (int)sizeof(T);  // bytes of a row
  static constexpr int NC = RB / 16;             // its chunks
  static constexpr int EC = 16 / (int)sizeof(T);
  static constexpr int NP = NC / 2;              // operands of a lane: every other chunk
  static constexpr int DT = D / 32;              // 32-channel tiles of the output
};

// Rows lie in LDS with chunk c at place c ^ swizzle(row): the 8 or 16 rows that
// one phase of an operand read touches, and the four rows of a transposing
// read, then lie in different banks (rows are 64, 128, 256 or 512 bytes).
template <int RB>
__device__ __forceinline__ int swizzle(int r) {
  if constexpr (RB >= 256) return ((r & 3) << 1) | ((r >> 2) & 1) | (((r ^ (r >> 3)) & 1) << 3);
  else if constexpr (RB == 128) return ((r & 2) << 1) | (((r ^ (r >> 3)) & 1) << 1) | ((r >> 2) & 1);
  else return ((r ^ (r >> 2)) & 2) | ((r >> 2) & 1);
}
template <int RB>
__device__ __forceinline__ int lds_chunk(int row, int chunk) {  // byte offset
  return row * RB + ((chunk ^ swizzle<RB>(row)) << 4);
}

// acc += A B over one chunk pair; lane: row / column lane & 31, the half's chunk.
template <typename T>
__device__ __forceinline__ void mma_chunk(f32x16& acc, const u32x4& a, const u32x4& b) {
  if constexpr (sizeof(T) == 2) {
    acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), acc, 0, 0, 0);
  } else {
    const f32x4_t x = __builtin_bit_cast(f32x4_t, a), y = __builtin_bit_cast(f32x4_t, b);
#pragma unroll
    for (int j = 0; j < 4; ++j) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(x[j], y[j], acc, 0, 0, 0);
  }
}

// o[dt] += V^T P^T over the 32 keys of the rows at v (LDS, swizzled), P^T in
// the scores' registers.
template <typename T, int D>
__device__ __forceinline__ void mma_values(f32x16 (&o)[D / 32], const char* v, int row0, const f32x16& s, int lane) {
  using G = Geo<T, D>;
  if constexpr (sizeof(T) == 2) {
    const int g = lane >> 4, i = lane & 15;
    const int key0 = row0 + 4 * (g >> 1) + (i >> 2);
    const int chunk = 2 * (g & 1) + ((i & 3) >> 1), within = 8 * (i & 1);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      bf16x8 p;
#pragma unroll
      for (int e = 0; e < 8; ++e) p[e] = static_cast<__bf16>(s[8 * j + e]);
      const int ra = key0 + 16 * j, rb = ra + 8;
#pragma unroll
      for (int dt = 0; dt < G::DT; ++dt) {
        const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)(v + lds_chunk<G::RB>(ra, 4 * dt + chunk) + within));
        const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)(v + lds_chunk<G::RB>(rb, 4 * dt + chunk) + within));
        const bf16x8 a = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, p, o[dt], 0, 0, 0);
      }
    }
  } else {
    const int half = lane >> 5, c = lane & 31;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int key = row0 + 8 * (r >> 2) + 4 * half + (r & 3);
#pragma unroll
      for (int dt = 0; dt < G::DT; ++dt) {
        const float a = *reinterpret_cast<const float*>(v + lds_chunk<G::RB>(key, 8 * dt + (c >> 2)) + 4 * (c & 3));
        o[dt] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, s[r], o[dt], 0, 0, 0);
      }
    }
  }
}

// The wave's other half's value at the same column, joined by f.
template <typename F>
__device__ __forceinline__ float join_halves(float x, F f) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return f(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// The numbers of a chunk that are not finite become zero; whether there were any.
template <typename T>
__device__ __forceinline__ bool clear_nonfinite(u32x4& x) {
  uint32_t w[4] = {x.x, x.y, x.z, x.w};
  bool any = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 2) {
      if ((w[i] & 0x7f80u) == 0x7f80u) { any = true; w[i] &= 0xffff0000u; }
      if ((w[i] & 0x7f800000u) == 0x7f800000u) { any = true; w[i] &= 0xffffu; }
    } else {
      if ((w[i] & 0x7f800000u) == 0x7f800000u) { any = true; w[i] = 0; }
    }
  }
  x = u32x4{w[0], w[1], w[2], w[3]};
  return any;
}

// A tile of M rows of one sequence.
struct Tile {
  SeqSpan span;
  int n, row0, rows;  // rows: of the sequence, from its first new token
  int first, last;    // positions of the tile's first and last row (negative: none)
  int keys;           // what the tile sees: last + 1, or 0
  int chunk;          // keys of a split
  bool direct;        // the sequence is not split: this workgroup has the whole softmax
};

__device__ __forceinline__ int split_chunk(const AttnParams& p, int len) {
  if (len <= p.whole) return p.whole;
  const int c = (len + p.splits - 1) / p.splits;
  return max(p.min_chunk, (c + kMinChunk - 1) / kMinChunk * kMinChunk);
}

// Tiles are numbered through the sequences with room for one that is not full
// each: sequence n's begin at floor(first row / M) + n, which holds ceil(rows /
// M) of them and needs no sum over the sequences before.
__host__ __device__ inline int64_t tile_bound(int64_t tokens, int64_t seqs, int64_t group, int M, bool packed) {
  return packed ? tokens * group / M + seqs + 1 : seqs * ((group + M - 1) / M);
}
// Tile `local` of M rows of sequence tile.n, whose span is given.
template <int M>
__device__ __forceinline__ bool fill_tile(const AttnParams& p, int local, const SeqSpan& span, Tile& tile) {
  const int group = (int)p.group.d;
  tile.span = span;
  const int64_t rows = (int64_t)tile.span.count * group, row0 = (int64_t)local * M;
  if (row0 >= rows) return false;
  tile.rows = (int)rows;
  tile.row0 = (int)row0;
  const int base = tile.span.len - tile.span.count;
  tile.first = base + (int)p.group.div((uint32_t)row0);
  tile.last = base + (int)p.group.div((uint32_t)min(rows - 1, row0 + M - 1));
  tile.keys = p.s.num_pages == 0 ? 0 : max(0, tile.last + 1);
  // the same in every lane, and in scalar registers once it is said
  const auto same = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
  tile.span = {same(tile.span.first), same(tile.span.count), same(tile.span.len)};
  tile.first = same(tile.first);
  tile.last = same(tile.last);
  tile.keys = same(tile.keys);
  tile.chunk = same(split_chunk(p, tile.span.len));
  tile.direct = tile.span.len <= tile.chunk;
  return true;
}
template <int M>
__device__ __forceinline__ bool find_tile(const AttnParams& p, int64_t t, Tile& tile) {
  const int group = (int)p.group.d;
  int local;
  if (M == 32 && p.s.cu && p.key_rows == 32) {  // one tile a sequence
    tile.n = (int)t;
    local = 0;
  } else if (p.s.cu) {
    const auto begin = [&](int n) -> int64_t {
      return (n == 0 ? 0 : (int64_t)clamp_int(p.s.cu[n], 0, p.s.num_tokens) * group / M) + n;
    };
    tile.n = wave_upper(p.s.num_seqs, t, begin);
    local = (int)(t - begin(tile.n));
  } else {
    const int per = (group + M - 1) / M;
    tile.n = (int)(t / per);
    local = (int)(t - (int64_t)tile.n * per);
  }
  return fill_tile<M>(p, local, seq_span(p.s, tile.n), tile);
}

// f over the wave's x.
template <typename F>
__device__ __forceinline__ int wave_join(int x, F f) {
  x = f(x, __builtin_amdgcn_update_dpp(0, x, 0xB1, 0xF, 0xF, false));   // quad [1,0,3,2]
  x = f(x, __builtin_amdgcn_update_dpp(0, x, 0x4E, 0xF, 0xF, false));   // quad [2,3,0,1]
  x = f(x, __builtin_amdgcn_update_dpp(0, x, 0x141, 0xF, 0xF, false));  // half-row mirror
  x = f(x, __builtin_amdgcn_update_dpp(0, x, 0x140, 0xF, 0xF, false));  // row mirror
  auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  x = f((int)r[0], (int)r[1]);
  r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return __builtin_amdgcn_readfirstlane(f((int)r[0], (int)r[1]));
}
__device__ __forceinline__ int wave_sum(int x) {
  return wave_join(x, [](int a, int b) { return a + b; });
}

// The t-th of the M-row tiles of sequences of more than key_rows rows, those
// with the most keys first: lane n has sequence n (fewer than 64).  A tile's
// level is its last row counted from the sequence's first position, in tiles;
// a sequence has one tile a level from lo up, so the tiles from a level up are
// counted by one sum over the wave, and the level of the t-th by bisection.  In
// the sequences' order instead the last long ones begin when the rest is nearly
// done: 13 prompts of 250 to 1,659 tokens 106 us, so 87.
template <int M>
__device__ __forceinline__ bool find_longest(const AttnParams& p, int t, Tile& tile) {
  const int lane = threadIdx.x & 63;
  int lo = 0, tiles = 0;
  SeqSpan span = {0, 0, 0};
  if (lane <= p.s.num_seqs) {
    span = seq_span(p.s, lane);
    const int64_t rows = (int64_t)span.count * p.group.d;
    if (rows > p.key_rows) tiles = (int)((rows + M - 1) / M);
    lo = (int)min((int64_t)max(0, span.len - span.count) * p.group.d / M, (int64_t)1 << 30);
  }
  if (t >= wave_sum(tiles)) return false;
  const auto from = [&](int level) { return wave_sum(clamp_int(lo + tiles - level, 0, tiles)); };
  int x = 0, y = wave_join(lo + tiles, [](int a, int b) { return max(a, b); });
  while (y - x > 1) {  // from(x) > t >= from(y)
    const int mid = x + (y - x) / 2;
    if (from(mid) > t) x = mid;
    else y = mid;
  }
  // of the level's tiles the (t - from(y))-th; the sum by all lanes, outside the condition
  const int place = t - from(y);
  const bool mine = (lo <= x) & (x < lo + tiles);
  const uint64_t at = __ballot(mine);
  tile.n = __builtin_ctzll(__ballot(mine & (__popcll(at & ((1ull << lane) - 1)) == place)));
  const auto its = [&](int v) { return __builtin_amdgcn_readlane(v, tile.n); };
  return fill_tile<M>(p, x - its(lo), {its(span.first), its(span.count), its(span.len)}, tile);
}

// One query row of a lane.
struct Row {
  int64_t index;  // token * q_heads + head
  int pos;        // its position; -1: sees nothing
  bool live;
};
template <typename T, int D>
__device__ __forceinline__ Row load_row(const AttnParams& p, const Tile& tile, int kvh, int r, int half,
                                        u32x4 (&q)[Geo<T, D>::NP]) {
  using G = Geo<T, D>;
  Row row;
  row.live = r < tile.rows;
  row.pos = -1;
  row.index = 0;
#pragma unroll
  for (int i = 0; i < G::NP; ++i) q[i] = u32x4{0, 0, 0, 0};
  if (row.live) {
    const int j = (int)p.group.div((uint32_t)r), g = r - j * (int)p.group.d;
    const int h = kvh * (int)p.group.d + g, t = tile.span.first + j;
    row.index = (int64_t)t * p.q_heads + h;
    row.pos = max(-1, tile.span.len - tile.span.count + j);
    const T* src = static_cast<const T*>(p.q) + t * p.q_stride + (int64_t)h * D + half * G::EC;
#pragma unroll
    for (int i = 0; i < G::NP; ++i) q[i] = *reinterpret_cast<const u32x4*>(src + 2 * i * G::EC);
    if (p.negate) {
      const uint32_t sign = sizeof(T) == 2 ? 0x80008000u : 0x80000000u;
#pragma unroll
      for (int i = 0; i < G::NP; ++i) q[i] ^= sign;
    }
  }
  return row;
}
// The queries arrive before the loop over the keys, and after the first keys are
// asked for: waits inside the loop would hold the keys that are on their way.
template <int N>
__device__ __forceinline__ void arrived(u32x4 (&q)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+v"(q[i]));
}

// A row's softmax while its keys pass.  m is their exact maximum, so the likeliest
// key's probability is 1, which BF16 holds.  Some row of a wave raises it, and all
// of a tile's outputs are rescaled, in nearly every tile of the first fifty:
// followed only where it has grown by more than 2^8, 2,048 tokens after 14,336 take
// 584 us and not 603, 13 prompts 84 and not 87, but that probability is then rounded
// with the others: the output's error against 64 bits is 0.0023 of its size, so
// 0.0020 (0.0017 is the output's own rounding).
template <int DT> struct Running {
  float m, l;  // maximum (base 2), and the sum over this half's keys
  f32x16 o[DT];
  __device__ __forceinline__ void init() {
    m = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[dt][r] = 0.f;
  }
  // scores of N tiles of keys -> their probabilities
  template <int N>
  __device__ __forceinline__ void step(f32x16 (&s)[N], float scale2) {
    float mx = s[0][0];
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[n][r]);
    mx = join_halves(mx, [](float a, float b) { return fmaxf(a, b); }) * scale2;
    if (__any(mx > m)) {
      const float mn = fmaxf(m, mx);
      const float a = exp2_fast(m - (mn == -INFINITY ? 0.f : mn));
      m = mn;
      l *= a;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[dt][r] *= a;
    }
    const float base = m == -INFINITY ? 0.f : m;
    float sum = 0.f;
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[n][r] = exp2_fast(__builtin_fmaf(s[n][r], scale2, -base));
        sum += s[n][r];
      }
    l += sum;
  }
};

__device__ __forceinline__ int key_of(int r, int half) { return 8 * (r >> 2) + 4 * half + (r & 3); }

// A row of the output.  A lane holds four channels of every eight; in BF16 the
// halves exchange theirs, eight channels for eight, and store 16 bytes.
template <typename T, int D>
__device__ __forceinline__ void store_row(T* dst, const f32x16 (&o)[D / 32], float f, int half) {
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt) {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int r = 0; r < 16; r += 8) {
        u32x4 x;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const auto pair = [&](int at) -> uint32_t {
            return __builtin_bit_cast(uint32_t, bf16x2{static_cast<__bf16>(o[dt][at] * f), static_cast<__bf16>(o[dt][at + 1] * f)});
          };
          const auto y = __builtin_amdgcn_permlane32_swap(pair(r + 2 * i), pair(r + 4 + 2 * i), false, false);
          x[i] = y[0];
          x[2 + i] = y[1];
        }
        *reinterpret_cast<u32x4*>(dst + 32 * dt + 2 * r + 8 * half) = x;
      }
    } else {
#pragma unroll
      for (int r = 0; r < 16; r += 4)
        *reinterpret_cast<f32x4_t*>(dst + 32 * dt + key_of(r, half)) =
            f32x4_t{o[dt][r] * f, o[dt][r + 1] * f, o[dt][r + 2] * f, o[dt][r + 3] * f};
    }
  }
}

// What values that are not finite add to the rows that see them (the products
// ran with zeros there, so that a row that does not see them stays what it is):
// key by key, a product of those values alone, which only lanes whose row sees
// the key take.  bad: the tile's keys with such values.
template <typename T, int D, int N>
__device__ __forceinline__ void add_nonfinite(f32x16 (&o)[D / 32], const f32x16 (&s)[N], uint64_t bad, const AttnParams& p,
                                              int n, int kvh, int key0, int pos, int lane) {
  const int half = lane >> 5;
  while (bad) {
    const int i = __builtin_ctzll(bad);
    bad &= bad - 1;
    int row;
    const int page = page_entry(p.s, n, key0 + i, &row);
    if (!page_exists(p.s, page)) continue;
    const T* v = static_cast<const T*>(p.v_pages) + page * p.v_page_stride + ((int64_t)row * p.kv_heads + kvh) * D;
    const int key_half = (i >> 2) & 1, key_r = 4 * ((i & 31) >> 3) + (i & 3);
    float pr = 0.f;  // the key's probability, in the lanes of its half
#pragma unroll
    for (int t = 0; t < N; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (t == i >> 5 && r == key_r) pr = s[t][r];
    const bool sees = key0 + i <= pos;
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt) {
      float x = io<T>::load(v + 32 * dt + (lane & 31));
      if (half != key_half || fabsf(x) < INFINITY) x = 0.f;
      f32x16 add;
#pragma unroll
      for (int r = 0; r < 16; ++r) add[r] = 0.f;
      if constexpr (sizeof(T) == 2) {
        const __bf16 z = static_cast<__bf16>(0.f);
        add = __builtin_amdgcn_mfma_f32_32x32x16_bf16(bf16x8{static_cast<__bf16>(x), z, z, z, z, z, z, z},
                                                      bf16x8{static_cast<__bf16>(pr), z, z, z, z, z, z, z}, add, 0, 0, 0);
      } else {
        add = __builtin_amdgcn_mfma_f32_32x32x2f32(x, pr, add, 0, 0, 0);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) o[dt][r] += sees ? add[r] : 0.f;
    }
  }
}

// ---------------------------------------------------------------------------
// Up to 32 rows a tile: the keys over the waves.
// ---------------------------------------------------------------------------
template <typename T, int D> struct KeysLds {
  static constexpr int OS = D + 4;  // floats between the rows of a wave's output
  static constexpr int kStage = kWaves * 32 * Geo<T, D>::RB, kJoin = kWaves * 32 * OS * 4;
  __align__(16) char buf[kStage > kJoin ? kStage : kJoin];
  float m[kWaves][32], l[kWaves][32];
};

template <typename T, int D>
__device__ __forceinline__ void attend_keys(const AttnParams& p, unsigned block, KeysLds<T, D>& lds) {
  using G = Geo<T, D>;
  constexpr int OS = KeysLds<T, D>::OS;
  char* s_buf = lds.buf;
  float (&s_m)[kWaves][32] = lds.m;
  float (&s_l)[kWaves][32] = lds.l;

  const int kvh = block % p.kv_heads;
  const unsigned rest = block / p.kv_heads;
  const int split = rest % p.splits;
  Tile tile;
  if (!find_tile<32>(p, rest / p.splits, tile)) return;
  if (p.s.cu && tile.rows > p.key_rows) return;  // the other form's
  const int k0 = split * tile.chunk, k1 = min(k0 + tile.chunk, tile.keys);
  if (split > 0 && (k0 >= tile.keys || tile.direct)) return;

  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int col = lane & 31, half = lane >> 5;
  char* sv = s_buf + w * 32 * G::RB;
  const int tiles = k1 > k0 ? (k1 - k0 + 31) / 32 : 0;
  const T* kb = static_cast<const T*>(p.k_pages) + (int64_t)kvh * D + half * G::EC;
  const T* vb = static_cast<const T*>(p.v_pages) + (int64_t)kvh * D + half * G::EC;
  const int row_stride = p.kv_heads * D;

  // the table's entry and the row of this lane's key of tile t: looked up a
  // tile ahead and read only where the keys are loaded, so that nothing waits
  const auto look = [&](int t, int& r) -> int { return page_entry(p.s, tile.n, min(k0 + 32 * t + col, k1 - 1), &r); };
  u32x4 k[G::NP], v[G::NP];
  bool here = false;  // this lane's key is there
  const auto load = [&](int t, int page, int r) {
    here = page_exists(p.s, page);
    const int64_t at = here ? page : 0, off = here ? (int64_t)r * row_stride : 0;
    here = here && k0 + 32 * t + col < k1;
    const T* ks = kb + at * p.k_page_stride + off;
    const T* vs = vb + at * p.v_page_stride + off;
#pragma unroll
    for (int i = 0; i < G::NP; ++i) k[i] = *reinterpret_cast<const u32x4*>(ks + 2 * i * G::EC);
#pragma unroll
    for (int i = 0; i < G::NP; ++i) v[i] = *reinterpret_cast<const u32x4*>(vs + 2 * i * G::EC);
  };

  int page = 0, r = 0;
  if (w < tiles) page = look(w, r);
  u32x4 q[G::NP];
  const Row row = load_row<T, D>(p, tile, kvh, tile.row0 + col, half, q);
  Running<G::DT> run;
  run.init();
  if (w < tiles) {
    int page1 = 0, r1 = 0;
    if (w + kWaves < tiles) page1 = look(w + kWaves, r1);
    load(w, page, r);
    page = page1;
    r = r1;
  }
  arrived(q);
  for (int t = w; t < tiles; t += kWaves) {
    const int key0 = k0 + 32 * t;
    const uint32_t there = (uint32_t)__ballot(here);
    f32x16 s[1];
#pragma unroll
    for (int r = 0; r < 16; ++r) s[0][r] = 0.f;
#pragma unroll
    for (int i = 0; i < G::NP; ++i) mma_chunk<T>(s[0], k[i], q[i]);
    // values to LDS: rows that are not there as zeros, and in a tile that some
    // row sees only part of, whatever is not finite
    const bool partial = key0 + 31 > tile.first;
    uint32_t bad = 0;
    if (there != 0xffffffffu) {
      if (!here)
#pragma unroll
        for (int i = 0; i < G::NP; ++i) v[i] = u32x4{0, 0, 0, 0};
    }
    if (partial && tile.first != tile.last) {
      bool any = false;
#pragma unroll
      for (int i = 0; i < G::NP; ++i) any |= clear_nonfinite<T>(v[i]);
      const uint64_t b = __ballot(any);
      bad = (uint32_t)b | (uint32_t)(b >> 32);
    }
#pragma unroll
    for (int i = 0; i < G::NP; ++i) *reinterpret_cast<u32x4*>(sv + lds_chunk<G::RB>(col, 2 * i + half)) = v[i];
    if (t + kWaves < tiles) {
      int page1 = 0, r1 = 0;
      if (t + 2 * kWaves < tiles) page1 = look(t + 2 * kWaves, r1);
      load(t + kWaves, page, r);
      page = page1;
      r = r1;
    }
    if (partial || there != 0xffffffffu) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int i = key_of(r, half);
        if (key0 + i > row.pos || !((there >> i) & 1)) s[0][r] = -INFINITY;
      }
    }
    run.step(s, p.scale2);
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    mma_values<T, D>(run.o, sv, 0, s[0], lane);
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    if (bad) add_nonfinite<T, D, 1>(run.o, s, bad, p, tile.n, kvh, key0, row.pos, lane);
  }

  // the waves' parts: a common maximum, then a sum over the waves in order
  const float l = join_halves(run.l, [](float a, float b) { return a + b; });
  if (half == 0) {
    s_m[w][col] = run.m;
    s_l[w][col] = l;
  }
  __syncthreads();
  const int live = min(32, tile.rows - tile.row0);
  {
    float m = s_m[0][col];
#pragma unroll
    for (int i = 1; i < kWaves; ++i) m = fmaxf(m, s_m[i][col]);
    const float a = exp2_fast(run.m - (m == -INFINITY ? 0.f : m));
    if (col < live) {
      float* so = reinterpret_cast<float*>(s_buf) + (w * 32 + col) * OS;
#pragma unroll
      for (int dt = 0; dt < G::DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; r += 4)
          *reinterpret_cast<float4*>(so + 32 * dt + key_of(r, half)) =
              make_float4(run.o[dt][r] * a, run.o[dt][r + 1] * a, run.o[dt][r + 2] * a, run.o[dt][r + 3] * a);
    }
  }
  __syncthreads();
  for (int x = threadIdx.x; x < live * (D / 4); x += kThreads) {
    const int i = x / (D / 4), c = 4 * (x % (D / 4));
    float m = s_m[0][i];
#pragma unroll
    for (int j = 1; j < kWaves; ++j) m = fmaxf(m, s_m[j][i]);
    float sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int j = 0; j < kWaves; ++j) {
      sum += s_l[j][i] * exp2_fast(s_m[j][i] - (m == -INFINITY ? 0.f : m));
      const float4 y = *reinterpret_cast<const float4*>(reinterpret_cast<float*>(s_buf) + (j * 32 + i) * OS + c);
      acc.x += y.x; acc.y += y.y; acc.z += y.z; acc.w += y.w;
    }
    const int r = tile.row0 + i, j = (int)p.group.div((uint32_t)r);
    const int64_t out = (int64_t)(tile.span.first + j) * p.q_heads + kvh * (int)p.group.d + (r - j * (int)p.group.d);
    if (tile.direct) {
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      store4(static_cast<T*>(p.o) + out * D + c, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
      if (c == 0) p.lse[out] = (m + __log2f(sum)) * 0.693147180559945309f;
    } else {
      const int64_t part = (int64_t)split * p.s.num_tokens * p.q_heads + out;
      *reinterpret_cast<float4*>(p.part_o + part * D + c) = acc;
      if (c == 0) *reinterpret_cast<float2*>(p.part_ml + part * 2) = make_float2(m, sum);
    }
  }
}

// ---------------------------------------------------------------------------
// More rows a sequence: 128 rows a tile over the waves, keys staged for all.
// ---------------------------------------------------------------------------
constexpr int kRowTile = 32 * kWaves;
constexpr int kKeyTile = 64;

// WHOLE: the rows that a wave stages at a time, 64 / NC keys, lie in one page
// (the page size is a multiple of them): a load's address is the page's, in
// scalar registers, and a lane's constant part.  2,048 tokens after 14,336:
// 603 us, with every lane's own addresses 645; 13 prompts: 87 and 91.
template <typename T, int D> struct RowsLds {
  __align__(16) char kv[4 * kKeyTile * Geo<T, D>::RB];  // two stages of K, V
  // of tile t % 3: its keys with values that are not finite, and those without a page
  __align__(16) uint32_t odd[3][4];
};

template <typename T, int D, bool WHOLE>
__device__ __forceinline__ void attend_rows(const AttnParams& p, unsigned block, RowsLds<T, D>& lds) {
  using G = Geo<T, D>;
  constexpr int NI = kKeyTile * G::NC / kThreads;  // chunks of K (and of V) a thread stages
  constexpr int RI = kThreads / G::NC;             // rows a pass of the workgroup covers
  constexpr int RW = 64 / G::NC;                   // and a wave of it
  constexpr int kTileBytes = kKeyTile * G::RB;
  char* s_kv = lds.kv;
  uint32_t (&s_odd)[3][4] = lds.odd;

  const int kvh = block % p.kv_heads;
  const unsigned rest = block / p.kv_heads;
  const int split = rest % p.splits;
  const int64_t bound = tile_bound(p.s.num_tokens, p.s.num_seqs, p.group.d, kRowTile, true);
  Tile tile;
  const int t = rest / p.splits;
  if (p.s.num_seqs < 64 ? !find_longest<kRowTile>(p, t, tile) : !find_tile<kRowTile>(p, bound - 1 - t, tile)) return;
  if (tile.rows <= p.key_rows) return;  // the other form's
  const int k0 = split * tile.chunk, k1 = min(k0 + tile.chunk, tile.keys);
  if (split > 0 && (k0 >= tile.keys || tile.direct)) return;

  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int col = lane & 31, half = lane >> 5;
  const int wrow0 = tile.row0 + 32 * w;
  // positions of the wave's first and last live row
  const int base = tile.span.len - tile.span.count;
  const bool wlive = wrow0 < tile.rows;
  const int wfirst = wlive ? base + (int)p.group.div((uint32_t)wrow0) : -1;
  const int wlast = wlive ? base + (int)p.group.div((uint32_t)min(tile.rows - 1, wrow0 + 31)) : -1;
  const int tiles = k1 > k0 ? (k1 - k0 + kKeyTile - 1) / kKeyTile : 0;
  const int srow = tid / G::NC, schunk = tid % G::NC;
  const int row_stride = p.kv_heads * D;
  // a lane's own part of an address: its chunk of its row of the wave's rows
  const uint32_t lane_off = (uint32_t)(WHOLE ? (srow - RW * w) * row_stride : 0) * sizeof(T) + schunk * 16;
  const char* kb = static_cast<const char*>(p.k_pages) + (int64_t)kvh * G::RB;
  const char* vb = static_cast<const char*>(p.v_pages) + (int64_t)kvh * G::RB;
  const int64_t k_page = p.k_page_stride * (int64_t)sizeof(T), v_page = p.v_page_stride * (int64_t)sizeof(T);

  // The table's entries of the next tile, looked up a tile ahead: of this thread's
  // rows, or (WHOLE) of the wave's, one a lane, so that all are found at once.
  constexpr int NL = WHOLE ? 1 : NI;
  int page[NL], prow[NL];
  const auto look = [&](int t) {
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int key = k0 + kKeyTile * t + (WHOLE ? RI * (lane & (NI - 1)) + RW * w : RI * i + srow);
      page[i] = page_entry(p.s, tile.n, min(key, WHOLE ? (k1 - 1) / RW * RW : k1 - 1), &prow[i]);
    }
  };
  u32x4 k[NI], v[NI];
  uint32_t gone = 0;  // this thread's staged rows that are not there, one bit each
  const auto load = [&](int t) {
    const char *ks[NI], *vs[NI];
    gone = 0;
    uint64_t ko[NL], vo[NL];
    bool here[NL];
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      here[i] = page_exists(p.s, page[i]);
      const uint32_t at = here[i] ? page[i] : 0, r = here[i] ? prow[i] : 0;
      const uint64_t off = (uint64_t)r * (uint32_t)(row_stride * (int)sizeof(T));
      ko[i] = at * (uint64_t)k_page + off;
      vo[i] = at * (uint64_t)v_page + off;
    }
    if constexpr (WHOLE) {
      const auto of_lane = [](uint64_t x, int i) {
        return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)x, i) |
               (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(x >> 32), i) << 32;
      };
      gone = ~(uint32_t)__ballot(here[0]) & ((1u << NI) - 1);
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        ks[i] = kb + of_lane(ko[0], i);
        vs[i] = vb + of_lane(vo[0], i);
      }
    } else {
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        gone |= (here[i] ? 0u : 1u) << i;
        ks[i] = kb + ko[i];
        vs[i] = vb + vo[i];
      }
    }
    if (t + 1 < tiles) look(t + 1);  // before the keys' loads, which it would otherwise wait for
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      k[i] = *reinterpret_cast<const u32x4*>(ks[i] + lane_off);
      v[i] = *reinterpret_cast<const u32x4*>(vs[i] + lane_off);
    }
    if (k0 + kKeyTile * (t + 1) > k1) {
#pragma unroll
      for (int i = 0; i < NI; ++i) gone |= (k0 + kKeyTile * t + srow + RI * i < k1 ? 0u : 1u) << i;
    }
  };
  const auto stage = [&](int t, int slot) {
    char* sk = s_kv + (t & 1) * 2 * kTileBytes;
    if (__any(gone)) {
#pragma unroll
      for (int i = 0; i < NI; ++i)
        if ((gone >> i) & 1) {
          const int r = RI * i + srow;
          v[i] = u32x4{0, 0, 0, 0};
          if (schunk == 0) atomicOr(&s_odd[slot][2 + (r >> 5)], 1u << (r & 31));
        }
    }
    if (k0 + kKeyTile * t + kKeyTile - 1 > tile.first) {
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int r = RI * i + srow;
        if (clear_nonfinite<T>(v[i])) atomicOr(&s_odd[slot][r >> 5], 1u << (r & 31));
      }
    }
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int at = lds_chunk<G::RB>(RI * i + srow, schunk);
      *reinterpret_cast<u32x4*>(sk + at) = k[i];
      *reinterpret_cast<u32x4*>(sk + kTileBytes + at) = v[i];
    }
  };
  if (tiles > 0) look(0);
  u32x4 q[G::NP];
  const Row row = load_row<T, D>(p, tile, kvh, wrow0 + col, half, q);
  Running<G::DT> run;
  run.init();
  if (tid < 12) s_odd[tid >> 2][tid & 3] = 0;
  if (tiles > 0) load(0);
  arrived(q);
  __syncthreads();
  if (tiles > 0) stage(0, 0);
  __syncthreads();
  int slot = 0;
  for (int t = 0; t < tiles; ++t) {
    const int key0 = k0 + kKeyTile * t, next = slot == 2 ? 0 : slot + 1, free = next == 2 ? 0 : next + 1;
    if (tid < 4) s_odd[free][tid] = 0;  // tile t + 2's, read last before the barrier that ended tile t - 1
    if (t + 1 < tiles) load(t + 1);
    const char* sk = s_kv + (t & 1) * 2 * kTileBytes;
    const u32x4 odd = *reinterpret_cast<const u32x4*>(s_odd[slot]);
    if (key0 <= wlast) {
      f32x16 s[2];
#pragma unroll
      for (int n = 0; n < 2; ++n) {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[n][r] = 0.f;
#pragma unroll
        for (int i = 0; i < G::NP; ++i) {
          const u32x4 a = *reinterpret_cast<const u32x4*>(sk + lds_chunk<G::RB>(32 * n + col, 2 * i + half));
          mma_chunk<T>(s[n], a, q[i]);
        }
      }
      const uint32_t gone0 = __builtin_amdgcn_readfirstlane(odd.z), gone1 = __builtin_amdgcn_readfirstlane(odd.w);
      if (key0 + kKeyTile - 1 > wfirst) {
        const int sees = row.pos - key0;  // the row sees keys up to this one of the tile
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (32 * n + key_of(r, half) > sees) s[n][r] = -INFINITY;
      }
      if (gone0 | gone1) {
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (((n ? gone1 : gone0) >> key_of(r, half)) & 1) s[n][r] = -INFINITY;
      }
      run.step(s, p.scale2);
#pragma unroll
      for (int n = 0; n < 2; ++n) mma_values<T, D>(run.o, sk + kTileBytes, 32 * n, s[n], lane);
      const uint64_t bad = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane(odd.x) |
                           (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane(odd.y) << 32;
      if (bad) add_nonfinite<T, D, 2>(run.o, s, bad, p, tile.n, kvh, key0, row.pos, lane);
    }
    if (t + 1 < tiles) stage(t + 1, next);
    slot = next;
    __syncthreads();
  }
  if (!row.live) return;
  const float l = join_halves(run.l, [](float a, float b) { return a + b; });
  if (tile.direct) {
    const float inv = l == 0.f ? 0.f : 1.f / l;
    store_row<T, D>(static_cast<T*>(p.o) + row.index * D, run.o, inv, half);
    if (half == 0) p.lse[row.index] = (run.m + __log2f(l)) * 0.693147180559945309f;
  } else {
    const int64_t part = (int64_t)split * p.s.num_tokens * p.q_heads + row.index;
    float* dst = p.part_o + part * D;
#pragma unroll
    for (int dt = 0; dt < G::DT; ++dt)
#pragma unroll
      for (int r = 0; r < 16; r += 4)
        *reinterpret_cast<float4*>(dst + 32 * dt + key_of(r, half)) =
            make_float4(run.o[dt][r], run.o[dt][r + 1], run.o[dt][r + 2], run.o[dt][r + 3]);
    if (half == 0) *reinterpret_cast<float2*>(p.part_ml + part * 2) = make_float2(run.m, l);
  }
}

// ---------------------------------------------------------------------------
template <typename T, int D, bool WHOLE>
__global__ __launch_bounds__(kThreads, (sizeof(T) == 4 && D == 128) ? 1 : 2) void paged_attention_kernel(AttnParams p) {
  __shared__ union Lds {
    KeysLds<T, D> keys;
    RowsLds<T, D> rows;
  } lds;
  if (blockIdx.x < p.row_blocks) attend_rows<T, D, WHOLE>(p, blockIdx.x, lds.rows);
  else attend_keys<T, D>(p, blockIdx.x - p.row_blocks, lds.keys);
}
// Without cu_seqlens every sequence has group rows and only the first form runs.
template <typename T, int D>
__global__ __launch_bounds__(kThreads, (sizeof(T) == 4 && D == 128) ? 1 : 2) void paged_attention_token_kernel(AttnParams p) {
  __shared__ KeysLds<T, D> lds;
  attend_keys<T, D>(p, blockIdx.x, lds);
}

// ---------------------------------------------------------------------------
// Joining the splits of a row: W waves a row, lanes over channels and parts.
// ---------------------------------------------------------------------------
template <typename T, int D, int W>
__global__ __launch_bounds__(kThreads) void paged_attention_join_kernel(AttnParams p) {
  constexpr int N = 64 * W;     // threads of a row
  constexpr int L = D / 4;      // threads of a part
  constexpr int PP = N / L;     // parts at a time
  constexpr int R = kThreads / N;
  __shared__ float4 s_acc[kThreads];
  __shared__ float s_w[R][kMaxSplits];
  const int64_t rows = (int64_t)p.s.num_tokens * p.q_heads;
  const int slot = W == kWaves ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / N);
  const int tid = threadIdx.x % N, lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * R + slot;
  bool mine = row < rows;
  const int t = mine ? (int)(row / p.q_heads) : 0;
  const int n = seq_of_token(p.s, t);
  const SeqSpan span = seq_span(p.s, n);
  const int j = t - span.first;
  const int chunk = split_chunk(p, span.len);
  // written already: rows of no sequence, and those of one that is not split
  mine = mine && n < p.s.num_seqs && (unsigned)j < (unsigned)span.count && span.len > chunk;
  const int pos = span.len - span.count + j;
  const int parts = !mine || pos < 0 || p.s.num_pages == 0 ? 0 : pos / chunk + 1;
  // every wave finds the row's maximum and sum for itself
  float m = -INFINITY;
  for (int i = lane; i < parts; i += 64) m = fmaxf(m, p.part_ml[(i * rows + row) * 2]);
#pragma unroll
  for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
  const float base = m == -INFINITY ? 0.f : m;
  float sum = 0.f;
  for (int i = lane; i < parts; i += 64) {
    const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + (i * rows + row) * 2);
    const float a = exp2_fast(ml.x - base);
    sum += ml.y * a;
    if (tid < 64) s_w[slot][i] = a;
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
  __syncthreads();
  const int x = tid / L, c = 4 * (tid % L);
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
  for (int i = x; i < parts; i += PP) {
    const float4 y = *reinterpret_cast<const float4*>(p.part_o + (i * rows + row) * D + c);
    const float a = s_w[slot][i];
    acc.x += y.x * a; acc.y += y.y * a; acc.z += y.z * a; acc.w += y.w * a;
  }
  s_acc[threadIdx.x] = acc;
  __syncthreads();
  if (x != 0 || !mine) return;
  for (int i = 1; i < PP; ++i) {
    const float4 y = s_acc[threadIdx.x + i * L];
    acc.x += y.x; acc.y += y.y; acc.z += y.z; acc.w += y.w;
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  store4(static_cast<T*>(p.o) + row * D + c, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
  if (c == 0) p.lse[row] = (m + __log2f(sum)) * 0.693147180559945309f;
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------
constexpr int64_t kSlots = 512;  // workgroups the card holds: two a compute unit

struct Plan {
  int64_t row_tiles, key_tiles;
};

// Which form takes which sequences, and into how many splits a sequence's keys
// are cut at most, from what the host knows: sequences have num_tokens /
// num_seqs tokens each.  Times are BF16, heads of 128, unless they say more.
Plan plan(AttnParams& p, bool packed) {
  const int64_t group = p.group.d, N = p.s.num_tokens, S = p.s.num_seqs, heads = p.kv_heads;
  Plan r;
  // More than 32 rows a sequence go to 128-row tiles: 13 prompts take 87 us so,
  // and 238 as tiles of 32 rows; 64 sequences of 40 rows after 1,900 keys 81 and
  // 101.  Not where those tiles leave the card half empty: one prompt of 1,531
  // tokens, 8/2 heads, is 98 of them (48 us) or 386 of 32 rows (36 us).
  p.key_rows = 32;
  r.row_tiles = packed ? tile_bound(N, S, group, kRowTile, true) : 0;
  if (packed && r.row_tiles * heads < kSlots / 2) p.key_rows = INT32_MAX;
  if (p.key_rows != 32) r.row_tiles = 0;
  r.key_tiles = packed && p.key_rows == 32 ? S + 1 : tile_bound(N, S, group, 32, packed);
  // A row's part of a split costs 2 D floats, a key 2 D numbers a tile: enough
  // keys a split that the parts stay a small share.  8 keys a row of the tile:
  // the 64 sequences of 40 rows take 81 us, with 16 they take 83.
  const int64_t per_seq = S > 0 && N > 0 ? (N * group + S - 1) / S : 1;
  const int64_t tile_rows = per_seq < 32 || p.key_rows != 32 ? (per_seq < 32 ? per_seq : 32)
                                                             : (per_seq < kRowTile ? per_seq : kRowTile);
  p.min_chunk = (int)((8 * tile_rows + kMinChunk - 1) / kMinChunk * kMinChunk);
  // Four times the workgroups the card holds where a sequence has less than a
  // full tile, since lengths differ and the longest decides: the same 64
  // sequences take 81 us with four, 89 with two, 127 with one.  Full tiles once:
  // their parts are many.
  const int64_t items = (packed && p.key_rows == 32 ? r.row_tiles + (per_seq <= 32 ? S : 0) : r.key_tiles) * heads;
  const int64_t cap = ((int64_t)p.s.max_pages * p.s.page_size + p.min_chunk - 1) / p.min_chunk;
  // Where the sequences fill the card by themselves, the short ones stay whole, and
  // all do where none can be long: 64 around 500 keys, 8 heads, take 29 us, and 38
  // in pieces; 128 around 1,000 120 and 126.  Longer ones differ by more than the
  // card evens out: 64 around 4,000, up to 7,500, 218 in four pieces and 296 whole
  // (228 with those up to 2,048 whole, 219 with those up to 1,024).
  p.whole = items >= kSlots ? 1024 : 0;
  int64_t want = kSlots * (per_seq < kRowTile ? 4 : 1) / (items > 0 ? items : 1);
  if ((int64_t)p.s.max_pages * p.s.page_size <= 2 * p.whole) want = 1;
  if (want > cap) want = cap;
  if (want > kMaxSplits) want = kMaxSplits;
  p.splits = want < 1 ? 1 : (int)want;
  return r;
}

template <typename T, int D>
int launch_attention(AttnParams p, hipStream_t s) {
  const Plan r = plan(p, p.s.cu != nullptr);
  const int64_t per_tile = (int64_t)p.kv_heads * p.splits;
  const int64_t blocks = (r.row_tiles + r.key_tiles) * per_tile;
  const int64_t rows = (int64_t)p.s.num_tokens * p.q_heads;
  PKDA_REQUIRE(blocks <= INT32_MAX && rows <= INT32_MAX, PKDA_EINVAL, "%d tokens of %d heads", p.s.num_tokens,
               p.q_heads);
  p.row_blocks = (unsigned)(r.row_tiles * per_tile);
  const dim3 grid((unsigned)blocks), block(kThreads);
  if (!p.s.cu)
    hipLaunchKernelGGL((paged_attention_token_kernel<T, D>), grid, block, 0, s, p);
  else if (p.s.page_size % (64 / Geo<T, D>::NC) == 0)
    hipLaunchKernelGGL((paged_attention_kernel<T, D, true>), grid, block, 0, s, p);
  else
    hipLaunchKernelGGL((paged_attention_kernel<T, D, false>), grid, block, 0, s, p);
  if (int st = launch_status("pkda_paged_attention")) return st;
  if (p.splits == 1) return 0;
  // A row's parts over four waves while rows are too few to fill the card: one
  // token after 131,071, 32 rows of 256 parts, 114 us against 120 in all; with
  // 10,240 rows of up to 10 parts one wave a row, 81 us against 95.
  if (rows < 2 * kSlots)
    hipLaunchKernelGGL((paged_attention_join_kernel<T, D, kWaves>), dim3((unsigned)rows), block, 0, s, p);
  else
    hipLaunchKernelGGL((paged_attention_join_kernel<T, D, 1>), dim3((unsigned)((rows + kWaves - 1) / kWaves)), block, 0, s, p);
  return launch_status("pkda_paged_attention(join)");
}

template <typename T>
int attention_dim(const AttnParams& p, int dim, hipStream_t s) {
  return dim == 128  ? launch_attention<T, 128>(p, s)
         : dim == 64 ? launch_attention<T, 64>(p, s)
                     : launch_attention<T, 32>(p, s);
}

int attention_sizes(const pkda_paged_attention_args* a, AttnParams& p) {
  PKDA_REQUIRE(a != nullptr, PKDA_EINVAL, "null args");
  PKDA_REQUIRE(a->struct_size == (int32_t)sizeof(*a), PKDA_EINVAL, "pkda_paged_attention_args size mismatch");
  if (int st = paged_seqs_from(a, p.s)) return st;
  PKDA_REQUIRE(a->q_heads >= 1 && a->q_heads <= 65535 && a->q_heads % a->kv_heads == 0, PKDA_EINVAL,
               "q_heads %d, kv_heads %d", a->q_heads, a->kv_heads);
  p.q_heads = a->q_heads;
  p.kv_heads = a->kv_heads;
  p.group = FastDiv::make((uint32_t)(a->q_heads / a->kv_heads));
  PKDA_REQUIRE((int64_t)a->num_tokens * p.group.d <= 1 << 30, PKDA_EINVAL, "%d tokens of %d heads", a->num_tokens,
               a->q_heads);
  plan(p, p.s.cu != nullptr);
  return 0;
}

}  // namespace
}  // namespace pkda

extern "C" int64_t pkda_paged_attention_workspace(const pkda_paged_attention_args* a) {
  pkda::AttnParams p;
  if (pkda::attention_sizes(a, p)) return -1;
  // by the sizes alone: one token a sequence may come with cu_seqlens or without
  pkda::plan(p, true);
  int splits = p.splits;
  if (a->num_tokens == a->num_seqs) {
    pkda::plan(p, false);
    splits = splits > p.splits ? splits : p.splits;
  }
  return splits > 1 ? (int64_t)splits * a->num_tokens * a->q_heads * (a->head_dim + 2) : 0;
}

extern "C" int pkda_paged_attention(const pkda_paged_attention_args* a, void* stream) {
  using namespace pkda;
  AttnParams p;
  if (int st = attention_sizes(a, p)) return st;
  const int64_t vec = a->dtype == PKDA_BF16 ? 8 : 4;
  if (int st = paged_pointers(a, vec)) return st;
  if (a->num_tokens == 0) return 0;
  PKDA_REQUIRE(a->q && a->o && a->lse, PKDA_EINVAL, "null tensor");
  PKDA_REQUIRE(a->q_stride % vec == 0 && ((uintptr_t)a->q | (uintptr_t)a->o) % 16 == 0, PKDA_EINVAL,
               "q and o must be 16-byte aligned");
  p.q = a->q; p.q_stride = a->q_stride; p.k_pages = a->k_pages; p.v_pages = a->v_pages;
  p.k_page_stride = a->k_page_stride; p.v_page_stride = a->v_page_stride;
  PKDA_REQUIRE(isfinite(a->scale), PKDA_EINVAL, "scale %g", (double)a->scale);
  // scale 0 as the smallest scale: a masked score stays -inf
  p.negate = a->scale < 0.f;
  p.scale2 = fmaxf(fabsf(a->scale) * kLog2e, 1e-37f);
  const int64_t rows = (int64_t)a->num_tokens * a->q_heads;
  PKDA_REQUIRE(p.splits == 1 || (a->workspace && (uintptr_t)a->workspace % 16 == 0), PKDA_EINVAL, "workspace");
  p.part_o = a->workspace;
  p.part_ml = a->workspace ? a->workspace + p.splits * rows * a->head_dim : nullptr;
  p.o = a->o; p.lse = a->lse;
  hipStream_t s = static_cast<hipStream_t>(stream);
  return a->dtype == PKDA_BF16 ? attention_dim<bf16_t>(p, a->head_dim, s) : attention_dim<float>(p, a->head_dim, s);
}
