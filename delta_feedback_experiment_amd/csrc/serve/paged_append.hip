// Appending new tokens' keys and values to a paged cache, with the rotary
// position embedding of queries and keys on the way (gfx950).
//
// Pairs (a, b) of the first rotary channels turn by their position's angle:
// a' = a cos - b sin, b' = b cos + a sin, in FP32, rounded once to the type.
//
// A pure copy by its bytes: q, k and v are read once, rotated q and the cache
// rows written once, one cos / sin row read a token.  A wave takes up to
// 2 * 64 / (D / 16) heads of one token, so that the token's sequence is
// searched once a wave (64 candidates a step), and a lane's cos and sin values
// serve every head it turns.  A lane owns 16 channels of a head: the two
// eight-channel vectors that rotate into each other, or two neighbouring ones
// past the rotated channels.  Every load of a lane goes out before its first
// use, and no lane writes what another reads: there is no LDS and no wait but
// for memory.
//
// Measured (BF16, heads of 128, every channel turned): 11,180 tokens of 16 + 2 x
// 4 heads in 13 sequences, 143 MB: 28 us (5.1 TB/s; a large copy runs at 4.8,
// and some of this stays in the last-level cache), with one head a lane at a
// time 29.3, with four 28.9; 4 tokens: 2.9 us, a launch and four trips to memory
// one after another (bounds, length, page, angles).
#include "paged_common.h"

namespace pkda {
namespace {

constexpr int kThreads = 256;
constexpr int kHeadsPerLane = 2;

struct AppendParams {
  PagedSeqs s;
  const void *q, *k, *v;
  int64_t q_stride, k_stride, v_stride;
  void *q_out, *k_pages, *v_pages;
  int64_t k_page_stride, v_page_stride;
  const float *cos, *sin;
  int q_heads, kv_heads, rotary, interleaved;
  int slots;  // waves of a token
};

template <typename T, int D>
__global__ __launch_bounds__(kThreads) void paged_append_kernel(AppendParams p) {
  constexpr int L = D / 16;   // lanes of a head
  constexpr int HW = 64 / L;  // heads of a wave at a time
  const int64_t wave = (int64_t)blockIdx.x * (kThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t tok = wave / p.slots;
  if (tok >= p.s.num_tokens) return;
  const int t = (int)tok, h0 = (int)(wave - tok * p.slots) * (HW * kHeadsPerLane);
  const int lane = threadIdx.x & 63, u = lane % L, hl = lane / L;

  // this lane's two vectors of a head, and which angles they turn by
  const int half = p.rotary / 2;
  const bool turns = 16 * u < p.rotary;
  const bool split = turns && !p.interleaved;
  const int c0 = split ? 8 * u : 16 * u, c1 = split ? 8 * u + half : 16 * u + 8;

  const int heads = p.q_heads + 2 * p.kv_heads;
  Vec8<T> x0[kHeadsPerLane], x1[kHeadsPerLane];
#pragma unroll
  for (int i = 0; i < kHeadsPerLane; ++i) {
    const int h = h0 + i * HW + hl;
    if (h >= heads) continue;
    const T* src;
    if (h < p.q_heads) src = static_cast<const T*>(p.q) + t * p.q_stride + (int64_t)h * D;
    else if (h < p.q_heads + p.kv_heads) src = static_cast<const T*>(p.k) + t * p.k_stride + (int64_t)(h - p.q_heads) * D;
    else src = static_cast<const T*>(p.v) + t * p.v_stride + (int64_t)(h - p.q_heads - p.kv_heads) * D;
    x0[i].load(src + c0);
    x1[i].load(src + c1);
  }

  const int n = seq_of_token(p.s, t);
  const SeqSpan span = seq_span(p.s, n);
  const int pos = span.len - span.count + (t - span.first);
  const bool placed = n < p.s.num_seqs && (unsigned)(t - span.first) < (unsigned)span.count && pos >= 0;
  int row = 0, page = -1;
  if (placed) {
    page = page_entry(p.s, n, pos, &row);
    if (!page_exists(p.s, page)) page = -1;
  }

  float cs[8], sn[8];
  if (turns && placed) {
    Vec8<float> c, s;
    c.load(p.cos + (int64_t)pos * half + 8 * u);
    s.load(p.sin + (int64_t)pos * half + 8 * u);
    c.get(cs);
    s.get(sn);
  }
  const int64_t row_off = (int64_t)row * p.kv_heads * D;
#pragma unroll
  for (int i = 0; i < kHeadsPerLane; ++i) {
    const int h = h0 + i * HW + hl;
    if (h >= heads) continue;
    const bool is_q = h < p.q_heads, is_v = h >= p.q_heads + p.kv_heads;
    if (turns && placed && !is_v) {
      float a[8], b[8], ya[8], yb[8];
      x0[i].get(a);
      x1[i].get(b);
      if (p.interleaved) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          ya[2 * j] = a[2 * j] * cs[j] - a[2 * j + 1] * sn[j];
          ya[2 * j + 1] = a[2 * j + 1] * cs[j] + a[2 * j] * sn[j];
          yb[2 * j] = b[2 * j] * cs[4 + j] - b[2 * j + 1] * sn[4 + j];
          yb[2 * j + 1] = b[2 * j + 1] * cs[4 + j] + b[2 * j] * sn[4 + j];
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          ya[j] = a[j] * cs[j] - b[j] * sn[j];
          yb[j] = b[j] * cs[j] + a[j] * sn[j];
        }
      }
      x0[i].set(ya);
      x1[i].set(yb);
    }
    T* dst;
    if (is_q) {
      if (!placed) {
        x0[i].zero();
        x1[i].zero();
      }
      dst = static_cast<T*>(p.q_out) + ((int64_t)t * p.q_heads + h) * D;
    } else {
      if (page < 0) continue;
      dst = is_v ? static_cast<T*>(p.v_pages) + page * p.v_page_stride + row_off + (int64_t)(h - p.q_heads - p.kv_heads) * D
                 : static_cast<T*>(p.k_pages) + page * p.k_page_stride + row_off + (int64_t)(h - p.q_heads) * D;
    }
    x0[i].store(dst + c0);
    x1[i].store(dst + c1);
  }
}

template <typename T, int D>
int launch_append(AppendParams p, hipStream_t s) {
  constexpr int per_wave = (64 / (D / 16)) * kHeadsPerLane;
  p.slots = (p.q_heads + 2 * p.kv_heads + per_wave - 1) / per_wave;
  const int64_t waves = (int64_t)p.s.num_tokens * p.slots;
  const int64_t blocks = (waves + kThreads / 64 - 1) / (kThreads / 64);
  PKDA_REQUIRE(blocks <= INT32_MAX, PKDA_EINVAL, "%d tokens of %d heads", p.s.num_tokens, p.q_heads + 2 * p.kv_heads);
  hipLaunchKernelGGL((paged_append_kernel<T, D>), dim3((unsigned)blocks), dim3(kThreads), 0, s, p);
  return launch_status("pkda_paged_append");
}

template <typename T>
int append_dim(const AppendParams& p, int dim, hipStream_t s) {
  return dim == 128 ? launch_append<T, 128>(p, s) : dim == 64 ? launch_append<T, 64>(p, s) : launch_append<T, 32>(p, s);
}

}  // namespace
}  // namespace pkda

extern "C" int pkda_paged_append(const pkda_paged_append_args* a, void* stream) {
  using namespace pkda;
  PKDA_REQUIRE(a != nullptr, PKDA_EINVAL, "null args");
  PKDA_REQUIRE(a->struct_size == (int32_t)sizeof(*a), PKDA_EINVAL, "pkda_paged_append_args size mismatch");
  AppendParams p;
  if (int st = paged_seqs_from(a, p.s)) return st;
  const int64_t vec = a->dtype == PKDA_BF16 ? 8 : 4;
  if (int st = paged_pointers(a, vec)) return st;
  PKDA_REQUIRE(a->q_heads >= 0 && a->q_heads <= 65535, PKDA_EINVAL, "q_heads %d", a->q_heads);
  PKDA_REQUIRE((a->cos == nullptr) == (a->sin == nullptr), PKDA_EINVAL, "cos without sin");
  const int rotary = a->cos ? a->rotary_dim : 0;
  PKDA_REQUIRE(rotary >= 0 && rotary <= a->head_dim && rotary % 16 == 0, PKDA_EUNSUPPORTED,
               "rotary_dim %d (a multiple of 16 up to head_dim %d)", rotary, a->head_dim);
  PKDA_REQUIRE(rotary == 0 || a->rope_rows >= (int64_t)a->max_pages * a->page_size, PKDA_EINVAL,
               "cos / sin hold %lld positions, a table row %lld", (long long)a->rope_rows,
               (long long)a->max_pages * a->page_size);
  if (a->num_tokens == 0) return 0;
  PKDA_REQUIRE(a->k && a->v && (a->q_heads == 0 || (a->q && a->q_out)), PKDA_EINVAL, "null tensor");
  PKDA_REQUIRE((a->k_stride | a->v_stride | (a->q_heads ? a->q_stride : 0)) % vec == 0 &&
                   ((uintptr_t)a->k | (uintptr_t)a->v | (uintptr_t)a->q | (uintptr_t)a->q_out | (uintptr_t)a->cos |
                    (uintptr_t)a->sin) % 16 == 0,
               PKDA_EINVAL, "q, k, v, cos, sin must be 16-byte aligned");
  p.q = a->q; p.k = a->k; p.v = a->v;
  p.q_stride = a->q_stride; p.k_stride = a->k_stride; p.v_stride = a->v_stride;
  p.q_out = a->q_out; p.k_pages = a->k_pages; p.v_pages = a->v_pages;
  p.k_page_stride = a->k_page_stride; p.v_page_stride = a->v_page_stride;
  p.cos = a->cos; p.sin = a->sin; p.q_heads = a->q_heads; p.kv_heads = a->kv_heads;
  p.rotary = rotary; p.interleaved = a->interleaved;
  hipStream_t s = static_cast<hipStream_t>(stream);
  return a->dtype == PKDA_BF16 ? append_dim<bf16_t>(p, a->head_dim, s) : append_dim<float>(p, a->head_dim, s);
}
