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
// 32 rows share tiles of 64 keys staged in LDS, double-buffered.  A third, the first
// in 16x16 tiles, takes one token a sequence of up to 16 rows, given without
// cu_seqlens, over an 8-bit cache and beside shared prefixes.  Where rows are
// few, a sequence's keys are split over workgroups and a second kernel joins the
// parts.
//
// Roundings to BF16: the probabilities, as the second product's operand (their
// sum l is of the unrounded ones), and the output; scores, m, l and O are FP32.
//
// What bounds it, measured in BF16 with heads of 128 (a large read runs at 4.0 to
// 5.0 TB/s, a large matrix product at 1188 TFLOP/s).  Decode, 256 sequences of
// 2,600 keys, 32/8 heads: 546 us, 4.98 TB/s of keys and values.  One sequence of
// 131,072 keys: 114 us, 4.7 TB/s.  2,048 tokens after 14,336, 32/8 heads: 595 to 624
// us by box, 825 to 865 TFLOP/s: a wave's 32 products a tile are 1,024 cycles, its 246 vector
// instructions, 32 exponentials among them, about 1,370, and its reads of LDS
// about 800; the other workgroup's wave on the SIMD overlaps them only in part
// (2,500 cycles a tile and wave).  13 prompts of 250 to 1,659 tokens, 16/4 heads:
// 86 to 92 us by box, 560 to 591 TFLOP/s: 6 us of a row tile's 33 are its way to its
// first keys and its output.
//
// Registers.  Of 256 a lane the 128-row form over an 8-bit cache, heads of 128, spills 7
// and reloads three of them in every tile of keys (4 and none where a wave's staged rows
// may lie in several pages; with shared prefixes it spills 6 and 3), and FP32 heads of 64
// spill up to 4.
#pragma once

#include <math.h>
#include <type_traits>

#include "paged_common.h"

namespace pkda {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kMaxSplits = 256;
constexpr int kMinChunk = 128;  // a split is a multiple of so many keys
constexpr int kRowTile = 32 * kWaves;
constexpr int kKeyTile = 64;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));
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
  // a cache of 8-bit floats: [num_pages][page_size][kv_heads][head_dim / 32] bytes
  const uint8_t *k_scales, *v_scales;
  int64_t k_scale_stride, v_scale_stride;
  // groups of sequences that share their first positions: sequences groups[g] ..
  // groups[g + 1] - 1 share prefix_lens[g]
  const int32_t *groups, *prefix_lens;
  int num_groups;
  bool ordered;  // attend_few: the longest sequences first
};

// What a workgroup attends: everything a sequence holds; or of a batch in groups
// the rows of a whole group over the positions that it shares, or a sequence's
// rows over the rest.
enum Part { kAll, kShared, kOwn };

// Rows of D channels as operands of type T, and as the cache stores them: the
// same, or 8-bit floats with a scale for each 32 channels.
template <typename T_, int D_, bool FP8_> struct Geo {
  using T = T_;
  static constexpr int D = D_;
  static constexpr bool FP8 = FP8_;
  static constexpr int RB = D * (int)sizeof(T);  // bytes of a row
  static constexpr int NC = RB / 16;             // its chunks
  static constexpr int EC = 16 / (int)sizeof(T);
  static constexpr int NP = NC / 2;              // operands of a lane
  static constexpr int DT = D / 32;              // 32-channel tiles of the output, scales of a row
  static constexpr int SB = FP8 ? D : RB;        // bytes of a stored row
  static constexpr int SC = SB / 16;             // its chunks
  static constexpr int SP = SC / 2;              // a lane's: every other chunk
  static constexpr int M = NC / SC;              // operands of a stored chunk
  static constexpr int ES = 16 * M / (int)sizeof(T);  // its channels
  // which chunk of a row operand i of a half is: the half's stored chunks' in turn
  __device__ __forceinline__ static int chunk(int i, int half) { return M * (2 * (i / M) + half) + i % M; }
};

// The operands of a stored chunk, whose scale is 2^(scale - 127): the product is
// exact in BF16 and in FP32.
template <typename G>
__device__ __forceinline__ void expand(const u32x4& x, uint32_t scale, u32x4* y) {
  if constexpr (!G::FP8) {
    y[0] = x;
  } else {
    const float f = __uint_as_float(scale << 23);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(typename G::T) == 2) {
        y[i / 2][2 * (i % 2)] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[i], f, false));
        y[i / 2][2 * (i % 2) + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[i], f, true));
      } else {
        const f32x2_t a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(x[i], f, false);
        const f32x2_t b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(x[i], f, true);
        y[i] = u32x4{__float_as_uint(a[0]), __float_as_uint(a[1]), __float_as_uint(b[0]), __float_as_uint(b[1])};
      }
    }
  }
}
// The scales of a row, a byte each.
template <int N>
__device__ __forceinline__ uint32_t load_scales(const uint8_t* p) {
  if constexpr (N == 4) return *reinterpret_cast<const uint32_t*>(p);
  else if constexpr (N == 2) return *reinterpret_cast<const uint16_t*>(p);
  else return *p;
}

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
// Of a row's chunk 0; that of chunk c differs by the bits of 16 c.  Eight rows on
// the swizzle has bit kFlip8 changed, and 16 rows on it is what it was.
template <int RB>
__device__ __forceinline__ int lds_row(int row) { return row * RB + (swizzle<RB>(row) << 4); }
template <int RB> constexpr int kFlip8 = RB >= 256 ? 8 : 2;
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
template <typename G>
__device__ __forceinline__ void mma_values(f32x16 (&o)[G::DT], const char* v, int row0, const f32x16& s, int lane) {
  using T = typename G::T;
  if constexpr (sizeof(T) == 2) {
    const int g = lane >> 4, i = lane & 15;
    const int key0 = row0 + 4 * (g >> 1) + (i >> 2);
    const int chunk = 2 * (g & 1) + ((i & 3) >> 1), within = 8 * (i & 1);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      bf16x8 p;
#pragma unroll
      for (int e = 0; e < 8; ++e) p[e] = static_cast<__bf16>(s[8 * j + e]);
      const auto add = [&](int dt, const char* at, const char* at8) {
        const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)at);
        const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)at8);
        const bf16x8 a = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, p, o[dt], 0, 0, 0);
      };
      if constexpr (G::FP8) {
        // Addresses of one register and the bits that differ.  A register each is 605
        // us for 2,048 tokens after 14,336 of a BF16 cache and so 613, but 626 of an
        // 8-bit cache and so 600.
        const int base = lds_row<G::RB>(key0) ^ (chunk << 4 | within);
#pragma unroll
        for (int dt = 0; dt < G::DT; ++dt)
          add(dt, v + 16 * j * G::RB + (base ^ (4 * dt << 4)),
              v + (16 * j + 8) * G::RB + (base ^ ((4 * dt ^ kFlip8<G::RB>) << 4)));
      } else {
        const int ra = key0 + 16 * j, rb = ra + 8;
#pragma unroll
        for (int dt = 0; dt < G::DT; ++dt)
          add(dt, v + lds_chunk<G::RB>(ra, 4 * dt + chunk) + within, v + lds_chunk<G::RB>(rb, 4 * dt + chunk) + within);
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
  int n, row0, rows;  // rows: of the sequence, from its first new token; n: whose pages
  int seq0, seq_end;  // kShared: the group's sequences are seq0 .. seq_end - 1
  int first, last;    // positions of the tile's first and last row (negative: none)
  int begin, keys;    // what the tile sees: positions begin .. keys - 1
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
// The positions that group g shares, those that whole tiles of keys hold: the
// others are each sequence's own, whose pages hold them too.
__device__ __forceinline__ int shared_len(const AttnParams& p, int g) {
  return (int)max((int64_t)0, min((int64_t)p.prefix_lens[g], (int64_t)p.s.max_pages * p.s.page_size)) / kKeyTile * kKeyTile;
}
__device__ __forceinline__ int group_bound(const AttnParams& p, int g) {
  return g == 0 ? 0 : clamp_int(p.groups[g], 0, p.s.num_seqs);
}
__device__ __forceinline__ int token_bound(const PagedSeqs& s, int n) {
  return n == 0 ? 0 : s.cu ? clamp_int(s.cu[n], 0, s.num_tokens) : n;
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

// A sequence of seq0 .. end - 1 that holds `want` positions, or where none does the
// longest: past its length a sequence's row of the table names nothing of its own (a
// slot that is finished is one of length 0), and none of the group's rows sees past
// the longest's.  By the whole wave.
__device__ __forceinline__ int holder_of(const PagedSeqs& s, int seq0, int end, int want) {
  const int lane = threadIdx.x & 63;
  int at = seq0, most = 0;
  for (int n = seq0; n < end; n += 64) {
    const int len = n + lane < end ? s.lens[n + lane] : -1;
    const uint64_t whole = __ballot(len >= want);
    if (whole) return n + __builtin_ctzll(whole);
    const int longest = wave_join(len, [](int a, int b) { return max(a, b); });
    if (longest > most) {
      most = longest;
      at = n + __builtin_ctzll(__ballot(len == longest));
    }
  }
  return at;
}
// The positions that sequence n shares with its group (none without one).
__device__ __forceinline__ int shared_of_seq(const AttnParams& p, int n) {
  const int g = wave_upper(p.num_groups, n, [&](int i) -> int64_t { return group_bound(p, i); });
  return g < p.num_groups ? shared_len(p, g) : 0;
}
// The position of token t, one of the new tokens of sequences n .. end - 1 (-1:
// it has none).  Each lane's own.
__device__ __forceinline__ int token_position(const PagedSeqs& s, int t, int n, int end) {
  if (!s.cu) return seq_span(s, t).len - 1;
  while (end - n > 1) {
    const int mid = n + (end - n) / 2;
    if (token_bound(s, mid) <= t) n = mid;
    else end = mid;
  }
  const SeqSpan span = seq_span(s, n);
  return t - span.first < span.count ? max(-1, span.len - span.count + (t - span.first)) : -1;
}

// Tile `local` of M rows of sequence tile.n, whose span is given (kShared: of a group
// of whose sequences it is one; len is what the group shares).
template <int M, Part PART = kAll>
__device__ __forceinline__ bool fill_tile(const AttnParams& p, int local, const SeqSpan& span, Tile& tile) {
  const int group = (int)p.group.d;
  tile.span = span;
  const int64_t rows = (int64_t)tile.span.count * group, row0 = (int64_t)local * M;
  if (row0 >= rows) return false;
  tile.rows = (int)rows;
  tile.row0 = (int)row0;
  tile.begin = 0;
  if constexpr (PART == kShared) {
    tile.first = tile.last = span.len - 1;  // rows that see less say so themselves
  } else {
    const int base = tile.span.len - tile.span.count;
    tile.first = base + (int)p.group.div((uint32_t)row0);
    tile.last = base + (int)p.group.div((uint32_t)min(rows - 1, row0 + M - 1));
  }
  tile.keys = p.s.num_pages == 0 ? 0 : max(0, tile.last + 1);
  // the same in every lane, and in scalar registers once it is said
  const auto same = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
  tile.span = {same(tile.span.first), same(tile.span.count), same(tile.span.len)};
  tile.first = same(tile.first);
  tile.last = same(tile.last);
  tile.keys = same(tile.keys);
  if constexpr (PART == kOwn) tile.begin = same(shared_of_seq(p, tile.n));
  tile.chunk = same(split_chunk(p, max(0, tile.span.len - tile.begin)));
  tile.direct = PART == kAll && tile.span.len <= tile.chunk;
  return true;
}
template <int M, Part PART = kAll>
__device__ __forceinline__ bool find_tile(const AttnParams& p, int64_t t, Tile& tile) {
  const int group = (int)p.group.d;
  int local;
  if constexpr (PART == kShared) {
    int g;
    const auto begin = [&](int i) -> int64_t {
      return (int64_t)token_bound(p.s, group_bound(p, i)) * group / M + i;
    };
    if (M == 32 && p.key_rows == 32) {  // one tile a group
      g = (int)t;
      local = 0;
    } else {
      g = wave_upper(p.num_groups, t, begin);
      local = (int)(t - begin(g));
    }
    if (g >= p.num_groups) return false;
    tile.seq0 = __builtin_amdgcn_readfirstlane(group_bound(p, g));
    tile.seq_end = __builtin_amdgcn_readfirstlane(group_bound(p, g + 1));
    if (tile.seq_end <= tile.seq0) return false;
    SeqSpan span;
    span.first = token_bound(p.s, tile.seq0);
    span.count = max(0, token_bound(p.s, tile.seq_end) - span.first);
    span.len = __builtin_amdgcn_readfirstlane(shared_len(p, g));
    tile.n = __builtin_amdgcn_readfirstlane(holder_of(p.s, tile.seq0, tile.seq_end, span.len));
    return fill_tile<M, kShared>(p, local, span, tile);
  }
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
  return fill_tile<M, PART>(p, local, seq_span(p.s, tile.n), tile);
}

// The t-th of the M-row tiles of sequences of more than key_rows rows, those
// with the most keys first: lane n has sequence n (fewer than 64).  A tile's
// level is its last row counted from the sequence's first position, in tiles;
// a sequence has one tile a level from lo up, so the tiles from a level up are
// counted by one sum over the wave, and the level of the t-th by bisection.  In
// the sequences' order instead the last long ones begin when the rest is nearly
// done: 13 prompts of 250 to 1,659 tokens 106 us, so 87.
template <int M, Part PART>
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
  return fill_tile<M, PART>(p, x - its(lo), {its(span.first), its(span.count), its(span.len)}, tile);
}

// One query row of a lane.
struct Row {
  int64_t index;  // token * q_heads + head
  int pos;        // its position; -1: sees nothing
  bool live;
};
template <typename G, Part PART>
__device__ __forceinline__ Row load_row(const AttnParams& p, const Tile& tile, int kvh, int r, int half,
                                        u32x4 (&q)[G::NP]) {
  using T = typename G::T;
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
    if constexpr (PART == kShared) row.pos = min(tile.last, token_position(p.s, t, tile.seq0, tile.seq_end));
    else row.pos = max(-1, tile.span.len - tile.span.count + j);
    const T* src = static_cast<const T*>(p.q) + t * p.q_stride + (int64_t)h * G::D;
#pragma unroll
    for (int i = 0; i < G::NP; ++i) q[i] = *reinterpret_cast<const u32x4*>(src + G::chunk(i, half) * G::EC);
    if (p.negate) {
      const uint32_t sign = sizeof(T) == 2 ? 0x80008000u : 0x80000000u;
#pragma unroll
      for (int i = 0; i < G::NP; ++i) q[i] ^= sign;
    }
  }
  return row;
}
// The queries arrive before the loop over the keys, and after the first keys are
// asked for: waits inside the loop would hold the keys that are on their way.  (A
// group's shared part asks for its keys after its rows' positions, whose lowest and
// highest it needs.)
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
template <typename G, int N>
__device__ __forceinline__ void add_nonfinite(f32x16 (&o)[G::DT], const f32x16 (&s)[N], uint64_t bad, const AttnParams& p,
                                              int n, int kvh, int key0, int pos, int lane) {
  using T = typename G::T;
  using S = std::conditional_t<G::FP8, uint8_t, T>;
  const int half = lane >> 5;
  while (bad) {
    const int i = __builtin_ctzll(bad);
    bad &= bad - 1;
    int row;
    const int page = page_entry(p.s, n, key0 + i, &row);
    if (!page_exists(p.s, page)) continue;
    const S* v = static_cast<const S*>(p.v_pages) + page * p.v_page_stride + ((int64_t)row * p.kv_heads + kvh) * G::D;
    const int key_half = (i >> 2) & 1, key_r = 4 * ((i & 31) >> 3) + (i & 3);
    float pr = 0.f;  // the key's probability, in the lanes of its half
#pragma unroll
    for (int t = 0; t < N; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (t == i >> 5 && r == key_r) pr = s[t][r];
    const bool sees = key0 + i <= pos;
#pragma unroll
    for (int dt = 0; dt < G::DT; ++dt) {
      float x;
      // (of the 8-bit floats only NaN is not finite)
      if constexpr (G::FP8) x = (v[32 * dt + (lane & 31)] & 0x7f) == 0x7f ? NAN : 0.f;
      else x = io<T>::load(v + 32 * dt + (lane & 31));
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
      __builtin_amdgcn_sched_barrier(0);  // one product's registers at a time: this is seldom run
    }
  }
}

// Which tile and split, and which key/value head, a workgroup of the keys' forms
// has.  Workgroups go to the eight dies in turn, each with an L2 of its own.  An
// 8-bit cache's scales of one head are 2 or 4 bytes of a line that holds the other
// heads' too, so there the heads of a tile are workgroups of one die: 256 sequences of 2,600
// keys, 8 heads, 291 us so and 365 with the heads over the dies.
struct Place {
  unsigned item;
  int head;
};
template <typename G>
__device__ __forceinline__ Place place_of(unsigned block, unsigned blocks, int heads) {
  if constexpr (G::FP8) {
    const unsigned round = 8u * heads, whole = blocks / round * round;
    if (block < whole) return {block / round * 8 + block % 8, (int)(block % round / 8)};
    const unsigned items = (blocks - whole) / heads;
    return {whole / heads + (block - whole) % items, (int)((block - whole) / items)};
  } else {
    return {block / heads, (int)(block % heads)};
  }
}

// ---------------------------------------------------------------------------
// Up to 32 rows a tile: the keys over the waves.
// ---------------------------------------------------------------------------
template <typename G> struct KeysLds {
  static constexpr int OS = G::D + 4;  // floats between the rows of a wave's output
  static constexpr int kStage = kWaves * 32 * G::RB, kJoin = kWaves * 32 * OS * 4;
  __align__(16) char buf[kStage > kJoin ? kStage : kJoin];
  float m[kWaves][32], l[kWaves][32];
};

template <typename G, Part PART>
__device__ __forceinline__ void attend_keys(const AttnParams& p, unsigned block, unsigned blocks, KeysLds<G>& lds) {
  using T = typename G::T;
  using S = std::conditional_t<G::FP8, uint8_t, T>;
  constexpr int D = G::D;
  constexpr int OS = KeysLds<G>::OS;
  char* s_buf = lds.buf;
  float (&s_m)[kWaves][32] = lds.m;
  float (&s_l)[kWaves][32] = lds.l;

  const auto [rest, kvh] = place_of<G>(block, blocks, p.kv_heads);
  const int split = rest % p.splits;
  Tile tile;
  if (!find_tile<32, PART>(p, rest / p.splits, tile)) return;
  if ((PART == kShared || p.s.cu) && tile.rows > p.key_rows) return;  // the other form's
  const int k0 = tile.begin + split * tile.chunk, k1 = min(k0 + tile.chunk, tile.keys);
  if (PART != kAll ? k0 >= tile.keys : split > 0 && (k0 >= tile.keys || tile.direct)) return;

  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int col = lane & 31, half = lane >> 5;
  char* sv = s_buf + w * 32 * G::RB;
  const int tiles = k1 > k0 ? (k1 - k0 + 31) / 32 : 0;
  const S* kb = static_cast<const S*>(p.k_pages) + (int64_t)kvh * D;
  const S* vb = static_cast<const S*>(p.v_pages) + (int64_t)kvh * D;
  const int row_stride = p.kv_heads * D;

  // the table's entry and the row of this lane's key of tile t: looked up a
  // tile ahead and read only where the keys are loaded, so that nothing waits
  const auto look = [&](int t, int& r) -> int { return page_entry(p.s, tile.n, min(k0 + 32 * t + col, k1 - 1), &r); };
  u32x4 k[G::SP], v[G::SP];
  uint32_t ks = 0, vs = 0;  // their scales
  bool here = false;        // this lane's key is there
  const auto load = [&](int t, int page, int r) {
    here = page_exists(p.s, page);
    const int64_t at = here ? page : 0, off = here ? (int64_t)r * row_stride : 0;
    const int64_t scale = G::FP8 ? off / 32 + kvh * G::DT : 0;
    here = here && k0 + 32 * t + col < k1;
    const S* kp = kb + (at * p.k_page_stride + off + half * G::ES);
    const S* vp = vb + (at * p.v_page_stride + off + half * G::ES);
    if constexpr (G::FP8) ks = load_scales<G::DT>(p.k_scales + at * p.k_scale_stride + scale);
#pragma unroll
    for (int i = 0; i < G::SP; ++i) k[i] = *reinterpret_cast<const u32x4*>(kp + 2 * i * G::ES);
    if constexpr (G::FP8) vs = load_scales<G::DT>(p.v_scales + at * p.v_scale_stride + scale);
#pragma unroll
    for (int i = 0; i < G::SP; ++i) v[i] = *reinterpret_cast<const u32x4*>(vp + 2 * i * G::ES);
  };

  int page = 0, r = 0;
  if (w < tiles) page = look(w, r);
  u32x4 q[G::NP];
  const Row row = load_row<G, PART>(p, tile, kvh, tile.row0 + col, half, q);
  if constexpr (PART == kShared)
    tile.first = wave_join(row.live ? row.pos : tile.last, [](int a, int b) { return min(a, b); });
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
  // this lane's row of operands in LDS: operand i is chunk(i, 0)'s bits away
  const int lrow = lds_row<G::RB>(col) ^ (G::chunk(0, half) << 4);
  for (int t = w; t < tiles; t += kWaves) {
    const int key0 = k0 + 32 * t;
    const uint32_t there = (uint32_t)__ballot(here);
    f32x16 s[1];
#pragma unroll
    for (int r = 0; r < 16; ++r) s[0][r] = 0.f;
#pragma unroll
    for (int i = 0; i < G::SP; ++i) {
      u32x4 x[G::M];
      expand<G>(k[i], (ks >> (8 * i)) & 0xff, x);
#pragma unroll
      for (int j = 0; j < G::M; ++j) mma_chunk<T>(s[0], x[j], q[G::M * i + j]);
    }
    // values to LDS: rows that are not there as zeros, and in a tile that some
    // row sees only part of, whatever is not finite
    const bool partial = key0 + 31 > tile.first;
    uint32_t bad = 0;
    if (there != 0xffffffffu) {
      if (!here) {
        vs = 0x7f7f7f7f;
#pragma unroll
        for (int i = 0; i < G::SP; ++i) v[i] = u32x4{0, 0, 0, 0};
      }
    }
    const bool clear = partial && tile.first != tile.last;
    bool any = false;
    if constexpr (G::FP8) {
#pragma unroll
      for (int i = 0; i < G::SP; ++i) {
        u32x4 x[G::M];
        expand<G>(v[i], (vs >> (8 * i)) & 0xff, x);
#pragma unroll
        for (int j = 0; j < G::M; ++j) {
          if (clear) any |= clear_nonfinite<T>(x[j]);
          *reinterpret_cast<u32x4*>(sv + (lrow ^ (G::chunk(G::M * i + j, 0) << 4))) = x[j];
        }
      }
    } else {
      if (clear) {
#pragma unroll
        for (int i = 0; i < G::NP; ++i) any |= clear_nonfinite<T>(v[i]);
      }
#pragma unroll
      for (int i = 0; i < G::NP; ++i) *reinterpret_cast<u32x4*>(sv + (lrow ^ (G::chunk(i, 0) << 4))) = v[i];
    }
    if (clear) {
      const uint64_t b = __ballot(any);
      bad = (uint32_t)b | (uint32_t)(b >> 32);
    }
    if (t + kWaves < tiles) {
      int page1 = 0, r1 = 0;
      if (t + 2 * kWaves < tiles) page1 = look(t + 2 * kWaves, r1);
      load(t + kWaves, page, r);
      page = page1;
      r = r1;
    }
    if (partial || there != 0xffffffffu) {
      const int sees = row.pos - key0 - 4 * half;  // of this half's keys, from its first on
      const uint32_t mine = there >> (4 * half);
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (key_of(r, 0) > sees || !((mine >> key_of(r, 0)) & 1)) s[0][r] = -INFINITY;
    }
    run.step(s, p.scale2);
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    mma_values<G>(run.o, sv, 0, s[0], lane);
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    if (bad) add_nonfinite<G, 1>(run.o, s, bad, p, tile.n, kvh, key0, row.pos, lane);
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
// One token a sequence and up to 16 query heads a key/value head: the keys over
// the waves, as above, in 16x16 MFMA tiles.  Half the registers and half the
// softmax's operations of the 32-row form, whose columns such a sequence does not
// fill: three workgroups a compute unit have keys on their way, and four query
// heads leave time for the conversions.  All rows are one token's: what a tile
// holds they all see.
// ---------------------------------------------------------------------------
template <typename G> struct FewLds {
  static constexpr int OS = G::D + 4;
  static constexpr int kStage = kWaves * 32 * G::RB, kJoin = kWaves * 16 * OS * 4;
  __align__(16) char buf[kStage > kJoin ? kStage : kJoin];
  float m[kWaves][16], l[kWaves][16];
};
constexpr int kFewRows = 16;

template <typename T>
__device__ __forceinline__ void mma_chunk16(f32x4_t& acc, const u32x4& a, const u32x4& b) {
  if constexpr (sizeof(T) == 2) {
    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), acc, 0, 0, 0);
  } else {
    const f32x4_t x = __builtin_bit_cast(f32x4_t, a), y = __builtin_bit_cast(f32x4_t, b);
#pragma unroll
    for (int j = 0; j < 4; ++j) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(x[j], y[j], acc, 0, 0, 0);
  }
}
// x of the four lanes of a column (lane & 15) joined by f.
template <typename F>
__device__ __forceinline__ float join_quarters(float x, F f) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return join_halves(f(__uint_as_float(r[0]), __uint_as_float(r[1])), f);
}

// The t-th longest of up to kOrdered sequences (ties by index), whose lengths the
// wave's lanes hold: by bisection over the length, the longer ones counted by
// ballots.
constexpr int kOrdered = 512;
__device__ __forceinline__ int longest_seq(const PagedSeqs& s, int t) {
  constexpr int N = kOrdered / 64;
  const int lane = threadIdx.x & 63, cap = s.max_pages * s.page_size;  // (at most 2^30)
  int len[N], hi = 0;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    len[j] = 64 * j + lane < s.num_seqs ? clamp_int(s.lens[64 * j + lane], 0, cap) : -1;
    hi = max(hi, len[j]);
  }
  const int sets = (s.num_seqs + 63) / 64;
  const auto count = [&](int x) {  // of that length and more
    int c = 0;
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j < sets) c += __popcll(__ballot(len[j] >= x));
    return c;
  };
  int lo = 0;
  hi = wave_join(hi, [](int a, int b) { return max(a, b); }) + 1;
  while (hi - lo > 1) {  // count(lo) > t >= count(hi)
    const int mid = lo + (hi - lo) / 2;
    if (count(mid) > t) lo = mid;
    else hi = mid;
  }
  int place = t - count(hi), n = 0;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const uint64_t at = __ballot(len[j] == lo);
    const int c = __popcll(at);
    if (place >= 0 && place < c)
      n = 64 * j + __builtin_ctzll(__ballot(len[j] == lo && __popcll(at & ((1ull << lane) - 1)) == place));
    place -= c;
  }
  return __builtin_amdgcn_readfirstlane(n);
}

template <typename G, Part PART>
__device__ __forceinline__ void attend_few(const AttnParams& p, unsigned block, unsigned blocks, FewLds<G>& lds) {
  using T = typename G::T;
  using S = std::conditional_t<G::FP8, uint8_t, T>;
  constexpr int D = G::D, CB = D / 16;   // 16-channel tiles of the output
  constexpr int LC = G::SC / 4;          // a lane's chunks of a key: every fourth
  constexpr int OS = FewLds<G>::OS;

  const auto [rest, kvh] = place_of<G>(block, blocks, p.kv_heads);
  const int split = rest % p.splits;
  Tile tile;
  // (group rows are one tile)
  tile.n = p.ordered ? longest_seq(p.s, (int)(rest / p.splits)) : (int)(rest / p.splits);
  fill_tile<kFewRows, PART>(p, 0, seq_span(p.s, tile.n), tile);
  const int k0 = tile.begin + split * tile.chunk, k1 = min(k0 + tile.chunk, tile.keys);
  if (PART != kAll ? k0 >= tile.keys : split > 0 && (k0 >= tile.keys || tile.direct)) return;

  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int col = lane & 15, g = lane >> 4;
  // Row m of a product's 16 keys is key `key`: bits 2 and 3 exchanged, so that the
  // rows which two quarters of a wave read at a time lie in different banks.
  const int key = ((col & 4) << 1) | ((col & 8) >> 1) | (col & 3), key4 = ((g & 1) << 3) | ((g & 2) << 1);
  char* sv = lds.buf + w * 32 * G::RB;
  const int tiles = k1 > k0 ? (k1 - k0 + 31) / 32 : 0;
  const S* kb = static_cast<const S*>(p.k_pages) + (int64_t)kvh * D;
  const S* vb = static_cast<const S*>(p.v_pages) + (int64_t)kvh * D;
  const int row_stride = p.kv_heads * D;

  u32x4 k[2][LC], v[2][LC];
  uint32_t ks[2] = {0, 0}, vs[2] = {0, 0};
  bool here[2] = {false, false};
  int page[2], prow[2];
  const auto look = [&](int t) {
#pragma unroll
    for (int b = 0; b < 2; ++b) page[b] = page_entry(p.s, tile.n, min(k0 + 32 * t + 16 * b + key, k1 - 1), &prow[b]);
  };
  const auto load = [&](int t) {
    int64_t ko[2], vo[2], kso[2], vso[2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      here[b] = page_exists(p.s, page[b]);
      const int64_t at = here[b] ? page[b] : 0, off = here[b] ? (int64_t)prow[b] * row_stride : 0;
      here[b] = here[b] && k0 + 32 * t + 16 * b + key < k1;
      ko[b] = at * p.k_page_stride + off + g * G::ES;
      vo[b] = at * p.v_page_stride + off + g * G::ES;
      if constexpr (G::FP8) {
        kso[b] = at * p.k_scale_stride + off / 32 + kvh * G::DT;
        vso[b] = at * p.v_scale_stride + off / 32 + kvh * G::DT;
      }
    }
    if (t + kWaves < tiles) look(t + kWaves);  // before the keys' loads, which it would otherwise wait for
    if constexpr (G::FP8) {
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        ks[b] = load_scales<G::DT>(p.k_scales + kso[b]);
        vs[b] = load_scales<G::DT>(p.v_scales + vso[b]);
      }
    }
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int j = 0; j < LC; ++j) k[b][j] = *reinterpret_cast<const u32x4*>(kb + ko[b] + 4 * j * G::ES);
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int j = 0; j < LC; ++j) v[b][j] = *reinterpret_cast<const u32x4*>(vb + vo[b] + 4 * j * G::ES);
  };
  // the scale of this lane's chunk j: a byte for two chunks
  const auto scale_of = [&](uint32_t scales, int j) { return (scales >> (8 * (2 * j + (g >> 1)))) & 0xff; };

  if (w < tiles) look(w);
  u32x4 q[LC][G::M];
#pragma unroll
  for (int j = 0; j < LC; ++j)
#pragma unroll
    for (int i = 0; i < G::M; ++i) {
      q[j][i] = u32x4{0, 0, 0, 0};
      if (col < tile.rows) {
        q[j][i] = *reinterpret_cast<const u32x4*>(static_cast<const T*>(p.q) + tile.span.first * p.q_stride +
                                                  (int64_t)(kvh * (int)p.group.d + col) * D + (G::M * (4 * j + g) + i) * G::EC);
        if (p.negate) q[j][i] ^= sizeof(T) == 2 ? 0x80008000u : 0x80000000u;
      }
    }
  float m = -INFINITY, l = 0.f;
  f32x4_t o[CB];
#pragma unroll
  for (int cb = 0; cb < CB; ++cb) o[cb] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  if (w < tiles) load(w);
#pragma unroll
  for (int j = 0; j < LC; ++j) arrived(q[j]);
  const int vrow = lds_row<G::RB>(key) ^ (G::M * g << 4);
  for (int t = w; t < tiles; t += kWaves) {
    uint32_t there[2];
#pragma unroll
    for (int b = 0; b < 2; ++b) there[b] = (uint32_t)__ballot(here[b]) >> (4 * g);  // of this quarter's keys, from bit 0 on
    f32x4_t s[2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      s[b] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < LC; ++j) {
        u32x4 x[G::M];
        expand<G>(k[b][j], scale_of(ks[b], j), x);
#pragma unroll
        for (int i = 0; i < G::M; ++i) mma_chunk16<T>(s[b], x[i], q[j][i]);
      }
    }
    const bool whole = __all(here[0] && here[1]);
    if (!whole) {
#pragma unroll
      for (int b = 0; b < 2; ++b)
        if (!here[b]) {
          vs[b] = 0x7f7f7f7f;
#pragma unroll
          for (int j = 0; j < LC; ++j) v[b][j] = u32x4{0, 0, 0, 0};
        }
    }
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int j = 0; j < LC; ++j) {
        u32x4 x[G::M];
        expand<G>(v[b][j], scale_of(vs[b], j), x);
#pragma unroll
        for (int i = 0; i < G::M; ++i)
          *reinterpret_cast<u32x4*>(sv + 16 * b * G::RB + (vrow ^ ((4 * G::M * j + i) << 4))) = x[i];
      }
    if (t + kWaves < tiles) load(t + kWaves);
    if (!whole) {
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (!((there[b] >> r) & 1)) s[b][r] = -INFINITY;
    }
    // the softmax's step, as in the other forms
    float mx = s[0][0];
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int r = 0; r < 4; ++r) mx = fmaxf(mx, s[b][r]);
    mx = join_quarters(mx, [](float a, float b) { return fmaxf(a, b); }) * p.scale2;
    if (__any(mx > m)) {
      const float mn = fmaxf(m, mx);
      const float a = exp2_fast(m - (mn == -INFINITY ? 0.f : mn));
      m = mn;
      l *= a;
#pragma unroll
      for (int cb = 0; cb < CB; ++cb)
#pragma unroll
        for (int r = 0; r < 4; ++r) o[cb][r] *= a;
    }
    const float base = m == -INFINITY ? 0.f : m;
    float sum = 0.f;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s[b][r] = exp2_fast(__builtin_fmaf(s[b][r], p.scale2, -base));
        sum += s[b][r];
      }
    l += sum;
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    if constexpr (sizeof(T) == 2) {
      bf16x8 pr;
#pragma unroll
      for (int e = 0; e < 8; ++e) pr[e] = static_cast<__bf16>(s[e >> 2][e & 3]);
      const int at = lds_row<G::RB>(key4 + (col >> 2)) ^ (((col & 3) >> 1) << 4 | 8 * (col & 1));
#pragma unroll
      for (int cb = 0; cb < CB; ++cb) {
        const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)(sv + (at ^ (2 * cb << 4))));
        const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)(sv + 16 * G::RB + (at ^ (2 * cb << 4))));
        const bf16x8 a = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        o[cb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, pr, o[cb], 0, 0, 0);
      }
    } else {
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int cb = 0; cb < CB; ++cb) {
            const float a = *reinterpret_cast<const float*>(sv + lds_chunk<G::RB>(16 * b + key4 + r, 4 * cb + (col >> 2)) + 4 * (col & 3));
            o[cb] = __builtin_amdgcn_mfma_f32_16x16x4f32(a, s[b][r], o[cb], 0, 0, 0);
          }
    }
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
  }

  // the waves' parts: a common maximum, then a sum over the waves in order
  l = join_quarters(l, [](float a, float b) { return a + b; });
  if (g == 0) {
    lds.m[w][col] = m;
    lds.l[w][col] = l;
  }
  __syncthreads();
  const int live = min(kFewRows, tile.rows);
  {
    float mx = lds.m[0][col];
#pragma unroll
    for (int i = 1; i < kWaves; ++i) mx = fmaxf(mx, lds.m[i][col]);
    const float a = exp2_fast(m - (mx == -INFINITY ? 0.f : mx));
    if (col < live) {
      float* so = reinterpret_cast<float*>(lds.buf) + (w * 16 + col) * OS + 4 * g;
#pragma unroll
      for (int cb = 0; cb < CB; ++cb)
        *reinterpret_cast<float4*>(so + 16 * cb) = make_float4(o[cb][0] * a, o[cb][1] * a, o[cb][2] * a, o[cb][3] * a);
    }
  }
  __syncthreads();
  for (int x = threadIdx.x; x < live * (D / 4); x += kThreads) {
    const int i = x / (D / 4), c = 4 * (x % (D / 4));
    float mx = lds.m[0][i];
#pragma unroll
    for (int j = 1; j < kWaves; ++j) mx = fmaxf(mx, lds.m[j][i]);
    float sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int j = 0; j < kWaves; ++j) {
      sum += lds.l[j][i] * exp2_fast(lds.m[j][i] - (mx == -INFINITY ? 0.f : mx));
      const float4 y = *reinterpret_cast<const float4*>(reinterpret_cast<float*>(lds.buf) + (j * 16 + i) * OS + c);
      acc.x += y.x; acc.y += y.y; acc.z += y.z; acc.w += y.w;
    }
    const int64_t out = (int64_t)tile.span.first * p.q_heads + kvh * (int)p.group.d + i;
    if (tile.direct) {
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      store4(static_cast<T*>(p.o) + out * D + c, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
      if (c == 0) p.lse[out] = (mx + __log2f(sum)) * 0.693147180559945309f;
    } else {
      const int64_t slot = (int64_t)split * p.s.num_tokens * p.q_heads + out;
      *reinterpret_cast<float4*>(p.part_o + slot * D + c) = acc;
      if (c == 0) *reinterpret_cast<float2*>(p.part_ml + slot * 2) = make_float2(mx, sum);
    }
  }
}

// ---------------------------------------------------------------------------
// More rows a sequence: 128 rows a tile over the waves, keys staged for all.
// ---------------------------------------------------------------------------
// WHOLE: the rows that a wave stages at a time, 64 / NC keys, lie in one page
// (the page size is a multiple of them): a load's address is the page's, in
// scalar registers, and a lane's constant part.  2,048 tokens after 14,336:
// 603 us, with every lane's own addresses 645; 13 prompts: 87 and 91.
template <typename G> struct RowsLds {
  __align__(16) char kv[4 * kKeyTile * G::RB];  // two stages of K, V
  // of tile t % 3: its keys with values that are not finite, and those without a page
  __align__(16) uint32_t odd[3][4];
  int first[kWaves];  // kShared: the lowest position of a wave's rows
};

template <typename G, bool WHOLE, Part PART>
__device__ __forceinline__ void attend_rows(const AttnParams& p, unsigned block, RowsLds<G>& lds) {
  using T = typename G::T;
  constexpr int D = G::D;
  constexpr int NI = kKeyTile * G::SC / kThreads;  // chunks of K (and of V) a thread stages
  constexpr int RI = kThreads / G::SC;             // rows a pass of the workgroup covers
  constexpr int RW = 64 / G::SC;                   // and a wave of it
  static_assert(NI >= 1, "a thread has a chunk to stage");
  constexpr int kTileBytes = kKeyTile * G::RB;
  char* s_kv = lds.kv;
  uint32_t (&s_odd)[3][4] = lds.odd;

  const int kvh = block % p.kv_heads;
  const unsigned rest = block / p.kv_heads;
  const int split = rest % p.splits;
  const int64_t bound = tile_bound(p.s.num_tokens, p.s.num_seqs, p.group.d, kRowTile, true);
  Tile tile;
  const int t = rest / p.splits;
  if constexpr (PART == kShared) {
    if (!find_tile<kRowTile, PART>(p, t, tile)) return;
  } else {
    if (p.s.num_seqs < 64 ? !find_longest<kRowTile, PART>(p, t, tile)
                          : !find_tile<kRowTile, PART>(p, bound - 1 - t, tile))
      return;
  }
  if (tile.rows <= p.key_rows) return;  // the other form's
  const int k0 = tile.begin + split * tile.chunk, k1 = min(k0 + tile.chunk, tile.keys);
  if (PART != kAll ? k0 >= tile.keys : split > 0 && (k0 >= tile.keys || tile.direct)) return;

  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int col = lane & 31, half = lane >> 5;
  const int wrow0 = tile.row0 + 32 * w;
  // positions of the wave's first and last live row
  const int base = tile.span.len - tile.span.count;
  const bool wlive = wrow0 < tile.rows;
  int wfirst = wlive ? base + (int)p.group.div((uint32_t)wrow0) : -1;
  int wlast = wlive ? base + (int)p.group.div((uint32_t)min(tile.rows - 1, wrow0 + 31)) : -1;
  const int tiles = k1 > k0 ? (k1 - k0 + kKeyTile - 1) / kKeyTile : 0;
  const int srow = tid / G::SC, schunk = tid % G::SC;
  const int row_stride = p.kv_heads * D;
  // a lane's own part of an address: its chunk of its row of the wave's rows
  constexpr int kItem = G::FP8 ? 1 : (int)sizeof(T);
  const uint32_t lane_off = (uint32_t)(WHOLE ? (srow - RW * w) * row_stride : 0) * kItem + schunk * 16;
  const char* kb = static_cast<const char*>(p.k_pages) + (int64_t)kvh * G::SB;
  const char* vb = static_cast<const char*>(p.v_pages) + (int64_t)kvh * G::SB;
  const int64_t k_page = p.k_page_stride * kItem, v_page = p.v_page_stride * kItem;
  // and of its scale's: a byte for two chunks
  const uint32_t lane_scale = (uint32_t)(WHOLE ? (srow - RW * w) * row_stride : 0) / 32 + kvh * G::DT + schunk / 2;

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
  uint32_t ksc[NI], vsc[NI];
  uint32_t gone = 0;  // this thread's staged rows that are not there, one bit each
  const auto load = [&](int t) {
    const char *ks[NI], *vs[NI];
    const uint8_t *kss[NI], *vss[NI];
    gone = 0;
    uint64_t ko[NL], vo[NL], kso[NL], vso[NL];
    bool here[NL];
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      here[i] = page_exists(p.s, page[i]);
      const uint32_t at = here[i] ? page[i] : 0, r = here[i] ? prow[i] : 0;
      const uint64_t off = (uint64_t)r * (uint32_t)(row_stride * kItem);
      ko[i] = at * (uint64_t)k_page + off;
      vo[i] = at * (uint64_t)v_page + off;
      if constexpr (G::FP8) {
        kso[i] = at * (uint64_t)p.k_scale_stride + off / 32;
        vso[i] = at * (uint64_t)p.v_scale_stride + off / 32;
      }
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
        if constexpr (G::FP8) {
          kss[i] = p.k_scales + of_lane(kso[0], i);
          vss[i] = p.v_scales + of_lane(vso[0], i);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        gone |= (here[i] ? 0u : 1u) << i;
        ks[i] = kb + ko[i];
        vs[i] = vb + vo[i];
        if constexpr (G::FP8) {
          kss[i] = p.k_scales + kso[i];
          vss[i] = p.v_scales + vso[i];
        }
      }
    }
    if (t + 1 < tiles) look(t + 1);  // before the keys' loads, which it would otherwise wait for
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      if constexpr (G::FP8) {
        ksc[i] = kss[i][lane_scale];
        vsc[i] = vss[i][lane_scale];
      }
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
          vsc[i] = 0x7f;
          if (schunk == 0) atomicOr(&s_odd[slot][2 + (r >> 5)], 1u << (r & 31));
        }
    }
    const bool clear = k0 + kKeyTile * t + kKeyTile - 1 > tile.first;
    if constexpr (G::FP8) {
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int r = RI * i + srow;
        u32x4 x[G::M], y[G::M];
        expand<G>(v[i], vsc[i], x);
        if (clear) {
          bool any = false;
#pragma unroll
          for (int j = 0; j < G::M; ++j) any |= clear_nonfinite<T>(x[j]);
          if (any) atomicOr(&s_odd[slot][r >> 5], 1u << (r & 31));
        }
        expand<G>(k[i], ksc[i], y);
#pragma unroll
        for (int j = 0; j < G::M; ++j) {
          const int at = lds_chunk<G::RB>(r, G::M * schunk + j);
          *reinterpret_cast<u32x4*>(sk + at) = y[j];
          *reinterpret_cast<u32x4*>(sk + kTileBytes + at) = x[j];
        }
      }
    } else {
      if (clear) {
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
    }
  };
  if (tiles > 0) look(0);
  u32x4 q[G::NP];
  const Row row = load_row<G, PART>(p, tile, kvh, wrow0 + col, half, q);
  if constexpr (PART == kShared) {
    wfirst = wave_join(row.live ? row.pos : tile.last, [](int a, int b) { return min(a, b); });
    wlast = wave_join(row.live ? row.pos : -1, [](int a, int b) { return max(a, b); });
    lds.first[w] = wfirst;
  }
  Running<G::DT> run;
  run.init();
  if (tid < 12) s_odd[tid >> 2][tid & 3] = 0;
  if (tiles > 0) load(0);
  arrived(q);
  __syncthreads();
  if constexpr (PART == kShared)
    tile.first = __builtin_amdgcn_readfirstlane(min(min(lds.first[0], lds.first[1]), min(lds.first[2], lds.first[3])));
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
          const u32x4 a = *reinterpret_cast<const u32x4*>(sk + lds_chunk<G::RB>(32 * n + col, G::chunk(i, half)));
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
      for (int n = 0; n < 2; ++n) mma_values<G>(run.o, sk + kTileBytes, 32 * n, s[n], lane);
      const uint64_t bad = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane(odd.x) |
                           (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane(odd.y) << 32;
      if (bad) add_nonfinite<G, 2>(run.o, s, bad, p, tile.n, kvh, key0, row.pos, lane);
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
template <typename G> union AttnLds {
  KeysLds<G> keys;
  RowsLds<G> rows;
};
// Workgroups of 256 registers a lane: two a compute unit, but for FP32 rows of 128.
template <typename G> constexpr int kPerUnit = sizeof(typename G::T) == 4 && G::D == 128 ? 1 : 2;

template <typename G, bool WHOLE>
__global__ __launch_bounds__(kThreads, kPerUnit<G>) void paged_attention_kernel(AttnParams p) {
  __shared__ AttnLds<G> lds;
  if (blockIdx.x < p.row_blocks) attend_rows<G, WHOLE, kAll>(p, blockIdx.x, lds.rows);
  else attend_keys<G, kAll>(p, blockIdx.x - p.row_blocks, gridDim.x - p.row_blocks, lds.keys);
}
// Without cu_seqlens every sequence has group rows and only the first form runs.
template <typename G>
__global__ __launch_bounds__(kThreads, kPerUnit<G>) void paged_attention_token_kernel(AttnParams p) {
  __shared__ KeysLds<G> lds;
  attend_keys<G, kAll>(p, blockIdx.x, gridDim.x, lds);
}
template <typename G>
__global__ __launch_bounds__(kThreads, sizeof(typename G::T) == 4 ? 2 : 3) void paged_attention_few_kernel(AttnParams p) {
  __shared__ FewLds<G> lds;
  attend_few<G, kAll>(p, blockIdx.x, gridDim.x, lds);
}
// A batch in groups: the groups' shared positions (their workgroups first, since
// they have the most keys), and the sequences' own.
// FEW: one token a sequence, of few query heads a key/value head.
template <typename G, bool WHOLE, bool FEW>
__global__ __launch_bounds__(kThreads, kPerUnit<G>) void paged_prefix_kernel(AttnParams shared, AttnParams own,
                                                                            unsigned shared_blocks) {
  __shared__ union {
    KeysLds<G> keys;
    RowsLds<G> rows;
    FewLds<G> few;
  } lds;
  if (blockIdx.x < shared_blocks) {
    if (blockIdx.x < shared.row_blocks) attend_rows<G, WHOLE, kShared>(shared, blockIdx.x, lds.rows);
    else attend_keys<G, kShared>(shared, blockIdx.x - shared.row_blocks, shared_blocks - shared.row_blocks, lds.keys);
  } else {
    const unsigned block = blockIdx.x - shared_blocks;
    if constexpr (FEW) {
      attend_few<G, kOwn>(own, block, gridDim.x - shared_blocks, lds.few);
    } else {
      if (block < own.row_blocks) attend_rows<G, WHOLE, kOwn>(own, block, lds.rows);
      else attend_keys<G, kOwn>(own, block - own.row_blocks, gridDim.x - shared_blocks - own.row_blocks, lds.keys);
    }
  }
}

// ---------------------------------------------------------------------------
// Joining the splits of a row: W waves a row, lanes over channels and parts.
// ---------------------------------------------------------------------------
// A row's parts: those of its sequence, or (GROUPS) those of its group's shared
// positions and then its sequence's own.
struct RowParts {
  int64_t rows, row;
  int shared;  // parts before the sequence's own
  int first;   // where those begin
  __device__ __forceinline__ int64_t at(int i) const { return (int64_t)(i < shared ? i : first + i - shared) * rows + row; }
};
template <typename T, int D, int W, bool GROUPS>
__global__ __launch_bounds__(kThreads) void paged_attention_join_kernel(AttnParams p, AttnParams own) {
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
  const int pos = span.len - span.count + j;
  RowParts at = {rows, row, 0, 0};
  int parts;
  if constexpr (GROUPS) {
    const int shared = shared_of_seq(p, n);
    const bool any = mine && n < p.s.num_seqs && (unsigned)j < (unsigned)span.count && pos >= 0 && p.s.num_pages > 0;
    const int own_chunk = split_chunk(own, max(0, span.len - shared));
    const int seen = min(shared, pos + 1), rest = pos + 1 - shared;
    if (any && shared > 0) at.shared = (seen - 1) / split_chunk(p, shared) + 1;
    at.first = p.splits;
    parts = at.shared + (any && rest > 0 ? (rest - 1) / own_chunk + 1 : 0);
  } else {
    const int chunk = split_chunk(p, span.len);
    // written already: rows of no sequence, and those of one that is not split
    mine = mine && n < p.s.num_seqs && (unsigned)j < (unsigned)span.count && span.len > chunk;
    parts = !mine || pos < 0 || p.s.num_pages == 0 ? 0 : pos / chunk + 1;
  }
  // every wave finds the row's maximum and sum for itself
  float m = -INFINITY;
  for (int i = lane; i < parts; i += 64) m = fmaxf(m, p.part_ml[at.at(i) * 2]);
#pragma unroll
  for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
  const float base = m == -INFINITY ? 0.f : m;
  float sum = 0.f;
  for (int i = lane; i < parts; i += 64) {
    const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + at.at(i) * 2);
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
    const float4 y = *reinterpret_cast<const float4*>(p.part_o + at.at(i) * D + c);
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
inline Plan plan(AttnParams& p, bool packed) {
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


// The longest sequences first where they do not all run at a time: 256 of 325 to
// 4,875 keys of an 8-bit cache, 8 heads, 297 us, in the caller's order 360 (all of
// one length: 291); 128 with 2 heads 52 and 49.
inline bool ordered(const AttnParams& p) {
  return p.s.num_seqs <= kOrdered && (int64_t)p.s.num_seqs * p.kv_heads >= kSlots;
}

// A row's parts over four waves while rows are too few to fill the card: one
// token after 131,071, 32 rows of 256 parts, 114 us against 120 in all; with
// 10,240 rows of up to 10 parts one wave a row, 81 us against 95.
template <typename G, bool GROUPS>
int launch_join(const AttnParams& p, const AttnParams& own, hipStream_t s, const char* what) {
  const int64_t rows = (int64_t)p.s.num_tokens * p.q_heads;
  const dim3 block(kThreads);
  if (rows < 2 * kSlots)
    hipLaunchKernelGGL((paged_attention_join_kernel<typename G::T, G::D, kWaves, GROUPS>), dim3((unsigned)rows), block, 0, s, p, own);
  else
    hipLaunchKernelGGL((paged_attention_join_kernel<typename G::T, G::D, 1, GROUPS>),
                       dim3((unsigned)((rows + kWaves - 1) / kWaves)), block, 0, s, p, own);
  return launch_status(what);
}

template <typename G>
int launch_attention(AttnParams p, hipStream_t s, const char* what) {
  const Plan r = plan(p, p.s.cu != nullptr);
  const int64_t per_tile = (int64_t)p.kv_heads * p.splits;
  const int64_t blocks = (r.row_tiles + r.key_tiles) * per_tile;
  const int64_t rows = (int64_t)p.s.num_tokens * p.q_heads;
  PKDA_REQUIRE(blocks <= INT32_MAX && rows <= INT32_MAX, PKDA_EINVAL, "%d tokens of %d heads", p.s.num_tokens,
               p.q_heads);
  p.row_blocks = (unsigned)(r.row_tiles * per_tile);
  const dim3 grid((unsigned)blocks), block(kThreads);
  if constexpr (G::FP8) {
    if (!p.s.cu && p.group.d <= kFewRows) {
      p.ordered = ordered(p);
      hipLaunchKernelGGL((paged_attention_few_kernel<G>), grid, block, 0, s, p);
      if (int st = launch_status(what)) return st;
      return p.splits == 1 ? 0 : launch_join<G, false>(p, p, s, what);
    }
  }
  if (!p.s.cu)
    hipLaunchKernelGGL((paged_attention_token_kernel<G>), grid, block, 0, s, p);
  else if (p.s.page_size % (64 / G::SC) == 0)
    hipLaunchKernelGGL((paged_attention_kernel<G, true>), grid, block, 0, s, p);
  else
    hipLaunchKernelGGL((paged_attention_kernel<G, false>), grid, block, 0, s, p);
  if (int st = launch_status(what)) return st;
  return p.splits == 1 ? 0 : launch_join<G, false>(p, p, s, what);
}

// What the attention entry points share.
template <typename A>
int attention_sizes(const A* a, AttnParams& p) {
  if (int st = paged_seqs_from(a, p.s)) return st;
  PKDA_REQUIRE(a->q_heads >= 1 && a->q_heads <= 65535 && a->q_heads % a->kv_heads == 0, PKDA_EINVAL,
               "q_heads %d, kv_heads %d", a->q_heads, a->kv_heads);
  p.q_heads = a->q_heads;
  p.kv_heads = a->kv_heads;
  p.group = FastDiv::make((uint32_t)(a->q_heads / a->kv_heads));
  PKDA_REQUIRE((int64_t)a->num_tokens * p.group.d <= 1 << 30, PKDA_EINVAL, "%d tokens of %d heads", a->num_tokens,
               a->q_heads);
  p.k_scales = p.v_scales = nullptr;
  p.k_scale_stride = p.v_scale_stride = 0;
  p.ordered = false;
  p.groups = p.prefix_lens = nullptr;
  p.num_groups = 0;
  plan(p, p.s.cu != nullptr);
  return 0;
}

// Floats of the parts of a call without groups.
template <typename A>
int64_t attention_workspace(const A* a, AttnParams p) {
  // by the sizes alone: one token a sequence may come with cu_seqlens or without
  plan(p, true);
  int splits = p.splits;
  if (a->num_tokens == a->num_seqs) {
    plan(p, false);
    splits = splits > p.splits ? splits : p.splits;
  }
  return splits > 1 ? (int64_t)splits * a->num_tokens * a->q_heads * (a->head_dim + 2) : 0;
}

// The tensors; parts: how many of each row the workspace holds.
template <typename A>
int attention_tensors(const A* a, AttnParams& p, int64_t vec, int parts) {
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
  PKDA_REQUIRE(parts == 1 || (a->workspace && (uintptr_t)a->workspace % 16 == 0), PKDA_EINVAL, "workspace");
  p.part_o = a->workspace;
  p.part_ml = a->workspace ? a->workspace + parts * rows * a->head_dim : nullptr;
  p.o = a->o; p.lse = a->lse;
  return 0;
}

}  // namespace
}  // namespace pkda
