// The paged key/value cache as the serving kernels see it (gfx950): which
// sequence and position a new token has, and where a position lies.
#pragma once

#include "pkda_common.h"
#include "serve/pkda_serve_gfx950.h"

namespace pkda {

// n / d for 0 <= n < 2^31, 1 <= d < 2^31, as a multiply and a shift: with
// s = ceil(log2 d) and m = ceil(2^(31+s) / d) < 2^32, m d - 2^(31+s) < d <= 2^s
// makes floor(n m / 2^(31+s)) exact (T. Granlund and P. Montgomery, "Division
// by invariant integers using multiplication", 1994).
struct FastDiv {
  uint32_t d, m, s;
  static FastDiv make(uint32_t d) {
    FastDiv f;
    f.d = d;
    f.s = 0;
    while ((uint64_t(1) << f.s) < d) ++f.s;
    f.m = static_cast<uint32_t>(((uint64_t(1) << (31 + f.s)) + d - 1) / d);
    return f;
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const {
    return static_cast<uint32_t>((static_cast<uint64_t>(n) * m) >> (31 + s));
  }
};

struct PagedSeqs {
  const int32_t* cu;     // [num_seqs + 1] or nullptr: one token a sequence
  const int32_t* lens;
  const int32_t* table;
  int64_t table_stride;
  int num_pages;
  int num_seqs, num_tokens;
  int page_size, max_pages;
  FastDiv page;
};

// One sequence: its new tokens [first, first + count) and its positions.
struct SeqSpan {
  int first, count, len;
};

__device__ __forceinline__ int clamp_int(int x, int lo, int hi) { return x < lo ? lo : (x > hi ? hi : x); }

// n <= num_seqs; num_seqs itself stands for the tokens past the last sequence,
// which have no positions.  Its loads are asked for together.
__device__ __forceinline__ SeqSpan seq_span(const PagedSeqs& s, int n) {
  if (!s.cu) {
    const int64_t cap = (int64_t)s.max_pages * s.page_size;
    return {n, 1, (int)max((int64_t)0, min((int64_t)s.lens[n], cap))};
  }
  if (s.num_seqs == 0) return {0, s.num_tokens, 0};
  const int m = min(n, s.num_seqs - 1);
  const int begin = s.cu[n], end = s.cu[m + 1], len = s.lens[m];
  SeqSpan r;
  r.first = n == 0 ? 0 : clamp_int(begin, 0, s.num_tokens);
  r.count = (n == s.num_seqs ? s.num_tokens : clamp_int(end, r.first, s.num_tokens)) - r.first;
  r.len = n == s.num_seqs ? 0 : (int)max((int64_t)0, min((int64_t)len, (int64_t)s.max_pages * s.page_size));
  return r;
}

// The largest n <= num_seqs with f(n) <= x, for f non-decreasing with
// f(0) <= x, by the whole wave, 64 candidates a step; x is wave-uniform.  Where
// f falls (bounds that cannot be) it is some n with f(n) <= x all the same: a
// step goes on from the last of the candidates before the first that is above.
template <typename F>
__device__ __forceinline__ int wave_upper(int num_seqs, int64_t x, F f) {
  const int lane = threadIdx.x & 63;
  int base = 0, span = num_seqs + 1;
  while (span > 1) {
    const int step = (span + 63) / 64;
    const int i = lane * step;
    const bool below = i < span && f(base + i) <= x;
    const uint64_t above = ~__ballot(below);
    const int at = (above ? __builtin_ctzll(above) - 1 : 63) * step;  // lane 0's is below
    base += at;
    span = min(step, span - at);
  }
  return __builtin_amdgcn_readfirstlane(base);
}

// The sequence of token t (num_seqs: of none).
__device__ __forceinline__ int seq_of_token(const PagedSeqs& s, int t) {
  if (!s.cu) return t;
  return wave_upper(s.num_seqs, t, [&](int n) -> int64_t {
    return n == 0 ? 0 : clamp_int(s.cu[n], 0, s.num_tokens);
  });
}

// What the table says of position p of sequence n (0 <= p < max_pages *
// page_size), and the position's row of that page.
__device__ __forceinline__ int page_entry(const PagedSeqs& s, int n, int p, int* row) {
  const int i = (int)s.page.div((uint32_t)p);
  *row = p - i * s.page_size;
  return s.table[(int64_t)n * s.table_stride + i];
}
// Whether the pool has such a page.
__device__ __forceinline__ bool page_exists(const PagedSeqs& s, int page) {
  return (uint32_t)page < (uint32_t)s.num_pages;
}

// Host: the arguments that append and attention share.
template <typename A>
int paged_seqs_from(const A* a, PagedSeqs& s) {
  PKDA_REQUIRE(a->dtype == PKDA_F32 || a->dtype == PKDA_BF16, PKDA_EUNSUPPORTED, "dtype %d", a->dtype);
  PKDA_REQUIRE(a->head_dim == 32 || a->head_dim == 64 || a->head_dim == 128, PKDA_EUNSUPPORTED,
               "head_dim %d (32, 64, 128)", a->head_dim);
  PKDA_REQUIRE(a->num_seqs >= 0 && a->num_tokens >= 0, PKDA_EINVAL, "num_seqs %d, num_tokens %d", a->num_seqs,
               a->num_tokens);
  PKDA_REQUIRE(a->kv_heads >= 1 && a->kv_heads <= 65535, PKDA_EINVAL, "kv_heads %d", a->kv_heads);
  // positions and a sequence's rows stay far enough under 2^31 that a tile past
  // the last one is still a number
  PKDA_REQUIRE(a->page_size >= 1 && a->max_pages >= 0 && (int64_t)a->page_size * a->max_pages <= 1 << 30,
               PKDA_EINVAL, "page_size %d x %d pages of a table row", a->page_size, a->max_pages);
  PKDA_REQUIRE(a->num_pages >= 0 && a->num_pages <= INT32_MAX, PKDA_EINVAL, "num_pages");
  s.cu = a->cu_seqlens; s.lens = a->seq_lens; s.table = a->page_table;
  s.table_stride = a->table_stride; s.num_pages = (int)a->num_pages;
  s.num_seqs = a->num_seqs; s.num_tokens = a->num_tokens;
  s.page_size = a->page_size; s.max_pages = a->max_pages;
  s.page = FastDiv::make((uint32_t)a->page_size);
  return 0;
}
template <typename A>
int paged_pointers(const A* a, int64_t vec) {  // vec: elements of 16 bytes
  PKDA_REQUIRE(a->cu_seqlens || a->num_tokens == a->num_seqs, PKDA_EINVAL,
               "%d tokens of %d sequences need cu_seqlens", a->num_tokens, a->num_seqs);
  PKDA_REQUIRE(a->seq_lens || a->num_seqs == 0, PKDA_EINVAL, "null seq_lens");
  PKDA_REQUIRE(a->page_table || (int64_t)a->num_seqs * a->max_pages == 0, PKDA_EINVAL, "null page_table");
  PKDA_REQUIRE(a->num_pages == 0 || (a->k_pages && a->v_pages), PKDA_EINVAL, "null pages");
  PKDA_REQUIRE((a->k_page_stride | a->v_page_stride) % vec == 0 &&
                   ((uintptr_t)a->k_pages | (uintptr_t)a->v_pages) % 16 == 0,
               PKDA_EINVAL, "pages must be 16-byte aligned");
  return 0;
}

}  // namespace pkda
