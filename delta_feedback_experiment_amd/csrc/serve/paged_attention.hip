// Attention of new tokens over a paged key/value cache (gfx950).
#include "paged_common.h"

namespace pkda {
namespace {

constexpr int kThreads = 256;

struct AttnParams {
  PagedSeqs s;
  const void* q;
  int64_t q_stride;
  const void *k_pages, *v_pages;
  int64_t k_page_stride, v_page_stride;
  int q_heads, kv_heads, group;
  float scale2;  // scale log2 e: the softmax is taken in base 2
  void* o;
  float* lse;
};

// One wave a (token, query head): a lane scores one of 64 positions, then owns
// D / 64 (at D = 32: one of 32) channels of the output.
template <typename T, int D>
__global__ __launch_bounds__(kThreads) void paged_attention_rows_kernel(AttnParams p) {
  __shared__ float s_q[kThreads / 64][D];
  __shared__ float s_p[kThreads / 64][64];
  __shared__ int64_t s_row[kThreads / 64][64];
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * (kThreads / 64) + w;
  const bool live = row < (int64_t)p.s.num_tokens * p.q_heads;
  const int t = live ? (int)(row / p.q_heads) : 0, h = live ? (int)(row - (int64_t)t * p.q_heads) : 0;
  if (!live) return;
  const int kvh = h / p.group;
  const int n = seq_of_token(p.s, t);
  const SeqSpan span = seq_span(p.s, n);
  const int j = t - span.first;
  const int last = n < p.s.num_seqs && (unsigned)j < (unsigned)span.count ? span.len - span.count + j : -1;
  for (int c = lane; c < D; c += 64) s_q[w][c] = io<T>::load(static_cast<const T*>(p.q) + t * p.q_stride + (int64_t)h * D + c);
  __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
  constexpr int NC = D < 64 ? 1 : D / 64;
  float acc[NC] = {}, m = -INFINITY, l = 0.f;
  for (int p0 = 0; p0 <= last; p0 += 64) {
    const int pos = p0 + lane;
    int r = 0, page = -1;
    if (pos <= last) page = page_of(p.s, n, pos, &r);
    float s = -INFINITY;
    const int64_t off = (int64_t)r * p.kv_heads * D + (int64_t)kvh * D;
    if (page >= 0) {
      const T* k = static_cast<const T*>(p.k_pages) + page * p.k_page_stride + off;
      float x = 0.f;
      for (int c = 0; c < D; ++c) x += s_q[w][c] * io<T>::load(k + c);
      s = x * p.scale2;
    }
    float mx = s;
#pragma unroll
    for (int o = 32; o; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
    const float mn = fmaxf(m, mx), base = mn == -INFINITY ? 0.f : mn;
    const float e = page >= 0 ? exp2_fast(s - base) : 0.f, a = exp2_fast(m - base);
    m = mn;
    float sum = e;
#pragma unroll
    for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
    l = l * a + sum;
    s_p[w][lane] = e;
    s_row[w][lane] = page >= 0 ? page * p.v_page_stride + off : -1;
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
#pragma unroll
    for (int i = 0; i < NC; ++i) acc[i] *= a;
    for (int i = 0; i < 64 && p0 + i <= last; ++i) {
      const int64_t at = s_row[w][i];
      if (at < 0) continue;
#pragma unroll
      for (int c = 0; c < NC; ++c)
        if (lane < D) acc[c] += s_p[w][i] * io<T>::load(static_cast<const T*>(p.v_pages) + at + c * 64 + lane);
    }
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int c = 0; c < NC; ++c)
    if (lane < D) io<T>::store(static_cast<T*>(p.o) + row * D + c * 64 + lane, acc[c] * inv);
  if (lane == 0) p.lse[row] = (m + __log2f(l)) * 0.693147180559945309f;
}

template <typename T, int D>
int launch_attention(const AttnParams& p, hipStream_t s) {
  const int64_t rows = (int64_t)p.s.num_tokens * p.q_heads;
  const int64_t blocks = (rows + kThreads / 64 - 1) / (kThreads / 64);
  PKDA_REQUIRE(blocks <= INT32_MAX, PKDA_EINVAL, "%lld rows", (long long)rows);
  hipLaunchKernelGGL((paged_attention_rows_kernel<T, D>), dim3((unsigned)blocks), dim3(kThreads), 0, s, p);
  return launch_status("pkda_paged_attention");
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
  p.group = a->q_heads / a->kv_heads;
  return 0;
}

}  // namespace
}  // namespace pkda

extern "C" int64_t pkda_paged_attention_workspace(const pkda_paged_attention_args* a) {
  pkda::AttnParams p;
  if (pkda::attention_sizes(a, p)) return -1;
  return 0;
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
  p.scale2 = a->scale * kLog2e;
  p.o = a->o; p.lse = a->lse;
  hipStream_t s = static_cast<hipStream_t>(stream);
  return a->dtype == PKDA_BF16 ? attention_dim<bf16_t>(p, a->head_dim, s) : attention_dim<float>(p, a->head_dim, s);
}
