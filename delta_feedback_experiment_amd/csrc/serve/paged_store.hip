// Appending new tokens' keys and values to a paged cache with the norms of query
// and key heads and the rotary position embedding on the way, into a cache of the
// activations' type or of 8-bit floats (gfx950).
//
// Per head, in FP32: x <- x (mean x^2 + eps)^(-1/2) w, then pairs (a, b) of the
// first rotary channels turn, a' = a cos - b sin, b' = b cos + a sin.  Into the
// activations' type that is rounded once.  Into 8-bit floats, blocks of 32
// channels take the smallest power of two s by which their largest magnitude is at
// most 448 (7/4 2^8, the largest code), and codes round x / s once, to the nearest;
// a power of two leaves the codes' relative error what it is for any scale, and
// code * s is a BF16 number.
//
// Bound by its bytes, as the plain append, whose layout of lanes it has: a wave
// takes up to 2 * 64 / (D / 16) heads of one token, a lane 16 channels of a head as
// two vectors of eight that rotate into each other (or neighbours).  A head's sum
// of squares is its D / 16 lanes'; a block's maximum too, block by block, since a
// lane's two vectors lie in blocks that depend on the rotated channels.
//
// Measured (BF16, heads of 128, every channel turned, norms): 11,180 tokens of 16 + 2
// x 4 heads in 13 sequences into 8-bit floats, 87 MB of least traffic: 20.7 us; into
// BF16, 94 MB: 20.3 us, 4.6 TB/s.  4 tokens: 3.7 us.
#include "paged_common.h"

namespace pkda {
namespace {

constexpr int kThreads = 256;
constexpr int kHeadsPerLane = 2;

struct StoreParams {
  PagedSeqs s;
  const void *q, *k, *v;
  int64_t q_stride, k_stride, v_stride;
  void *q_out, *k_pages, *v_pages;
  int64_t k_page_stride, v_page_stride;
  const float *cos, *sin;
  int q_heads, kv_heads, rotary, interleaved;
  int slots;  // waves of a token
  const void *q_norm, *k_norm;
  int norm_bf16;
  float eps;
  uint8_t *k_scales, *v_scales;
  int64_t k_scale_stride, v_scale_stride;
};

// The largest over each aligned group of N lanes of numbers >= 0, every lane of
// the group getting it.
template <int N>
__device__ __forceinline__ uint32_t lane_group_max(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, false));  // quad [1,0,3,2]
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, false));  // quad [2,3,0,1]
  if constexpr (N == 8) v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xF, 0xF, false));  // half-row mirror
  return v;
}

// The magnitude's bits, which are ordered as the magnitudes are; 0 for what is
// not finite.
__device__ __forceinline__ uint32_t finite_magnitude(float x) {
  const uint32_t b = __float_as_uint(x) & 0x7fffffffu;
  return b < 0x7f800000u ? b : 0;
}
// The exponent byte e of the smallest scale 2^(e - 127) of 2^-117 .. 2^119 by
// which a magnitude is at most 7/4 2^8.
__device__ __forceinline__ uint32_t scale_byte(uint32_t magnitude) {
  const int e = (int)(magnitude >> 23) - 8 + ((magnitude & 0x7fffffu) > 0x600000u ? 1 : 0);
  return (uint32_t)clamp_int(e, 10, 246);
}
// Eight numbers as codes; inv = 1 / scale.
__device__ __forceinline__ uint2 encode8(const float (&x)[8], float inv) {
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    y[i] = __builtin_amdgcn_fmed3f(x[i] * inv, -448.f, 448.f);
    if (!(fabsf(x[i]) < INFINITY)) y[i] = NAN;
  }
  int lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], lo, true);
  int hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[4], y[5], 0, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[6], y[7], hi, true);
  return make_uint2((uint32_t)lo, (uint32_t)hi);
}

template <typename T, int D, bool FP8>
__global__ __launch_bounds__(kThreads) void paged_store_kernel(StoreParams p) {
  constexpr int L = D / 16;   // lanes of a head
  constexpr int HW = 64 / L;  // heads of a wave at a time
  constexpr int NB = D / 32;  // its blocks
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
#pragma unroll
  for (int i = 0; i < kHeadsPerLane; ++i) {
    const int h = h0 + i * HW + hl;
    if (h >= heads) continue;  // (the lanes of a head go together)
    const bool is_q = h < p.q_heads, is_v = h >= p.q_heads + p.kv_heads;
    if (!is_q && page < 0) continue;
    float a[8], b[8];
    x0[i].get(a);
    x1[i].get(b);
    const void* weight = is_q ? p.q_norm : is_v ? nullptr : p.k_norm;
    if (weight) {
      float squares = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) squares += a[j] * a[j] + b[j] * b[j];
      squares = lane_group_sum<L>(squares);
      const float r = 1.f / sqrtf(squares * (1.f / D) + p.eps);
      float wa[8], wb[8];
      if (p.norm_bf16) {
        Vec8<bf16_t> w;
        w.load(static_cast<const bf16_t*>(weight) + c0);
        w.get(wa);
        w.load(static_cast<const bf16_t*>(weight) + c1);
        w.get(wb);
      } else {
        Vec8<float> w;
        w.load(static_cast<const float*>(weight) + c0);
        w.get(wa);
        w.load(static_cast<const float*>(weight) + c1);
        w.get(wb);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        a[j] = a[j] * r * wa[j];
        b[j] = b[j] * r * wb[j];
      }
    }
    const bool turned = turns && placed && !is_v;
    if (turned) {
      if (p.interleaved) {
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          const float a0 = a[j], a1 = a[j + 1], b0 = b[j], b1 = b[j + 1];
          a[j] = a0 * cs[j / 2] - a1 * sn[j / 2];
          a[j + 1] = a1 * cs[j / 2] + a0 * sn[j / 2];
          b[j] = b0 * cs[4 + j / 2] - b1 * sn[4 + j / 2];
          b[j + 1] = b1 * cs[4 + j / 2] + b0 * sn[4 + j / 2];
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float a0 = a[j], b0 = b[j];
          a[j] = a0 * cs[j] - b0 * sn[j];
          b[j] = b0 * cs[j] + a0 * sn[j];
        }
      }
    }
    const int kvh = is_v ? h - p.q_heads - p.kv_heads : h - p.q_heads;
    const int64_t at = ((int64_t)row * p.kv_heads + kvh) * D;
    if constexpr (FP8) {
      if (!is_q) {
        uint32_t ma = 0, mb = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          ma = max(ma, finite_magnitude(a[j]));
          mb = max(mb, finite_magnitude(b[j]));
        }
        const int ba = c0 / 32, bb = c1 / 32;
        uint32_t scales = 0, ea = 0, eb = 0;
#pragma unroll
        for (int j = 0; j < NB; ++j) {
          const uint32_t e = scale_byte(lane_group_max<L>(max(ba == j ? ma : 0u, bb == j ? mb : 0u)));
          scales |= e << (8 * j);
          if (ba == j) ea = e;
          if (bb == j) eb = e;
        }
        uint8_t* dst = static_cast<uint8_t*>(is_v ? p.v_pages : p.k_pages) + page * (is_v ? p.v_page_stride : p.k_page_stride) + at;
        *reinterpret_cast<uint2*>(dst + c0) = encode8(a, __uint_as_float((254 - ea) << 23));
        *reinterpret_cast<uint2*>(dst + c1) = encode8(b, __uint_as_float((254 - eb) << 23));
        if (u == 0) {
          uint8_t* sc = (is_v ? p.v_scales : p.k_scales) + page * (is_v ? p.v_scale_stride : p.k_scale_stride) + at / 32;
          if constexpr (NB == 4) *reinterpret_cast<uint32_t*>(sc) = scales;
          else *reinterpret_cast<uint16_t*>(sc) = (uint16_t)scales;
        }
        continue;
      }
    }
    if (weight || turned) {  // (what is only moved keeps its bits)
      x0[i].set(a);
      x1[i].set(b);
    }
    T* dst;
    if (is_q) {
      if (!placed) {
        x0[i].zero();
        x1[i].zero();
      }
      dst = static_cast<T*>(p.q_out) + ((int64_t)t * p.q_heads + h) * D;
    } else {
      dst = static_cast<T*>(is_v ? p.v_pages : p.k_pages) + page * (is_v ? p.v_page_stride : p.k_page_stride) + at;
    }
    x0[i].store(dst + c0);
    x1[i].store(dst + c1);
  }
}

template <typename T, int D, bool FP8>
int launch_store(StoreParams p, hipStream_t s) {
  constexpr int per_wave = (64 / (D / 16)) * kHeadsPerLane;
  p.slots = (p.q_heads + 2 * p.kv_heads + per_wave - 1) / per_wave;
  const int64_t waves = (int64_t)p.s.num_tokens * p.slots;
  const int64_t blocks = (waves + kThreads / 64 - 1) / (kThreads / 64);
  PKDA_REQUIRE(blocks <= INT32_MAX, PKDA_EINVAL, "%d tokens of %d heads", p.s.num_tokens, p.q_heads + 2 * p.kv_heads);
  hipLaunchKernelGGL((paged_store_kernel<T, D, FP8>), dim3((unsigned)blocks), dim3(kThreads), 0, s, p);
  return launch_status("pkda_paged_store");
}

template <typename T>
int store_dim(const StoreParams& p, int dim, bool fp8, hipStream_t s) {
  if (fp8) return dim == 128 ? launch_store<T, 128, true>(p, s) : launch_store<T, 64, true>(p, s);
  return dim == 128  ? launch_store<T, 128, false>(p, s)
         : dim == 64 ? launch_store<T, 64, false>(p, s)
                     : launch_store<T, 32, false>(p, s);
}

}  // namespace
}  // namespace pkda

extern "C" int pkda_paged_store(const pkda_paged_store_args* a, void* stream) {
  using namespace pkda;
  PKDA_REQUIRE(a != nullptr, PKDA_EINVAL, "null args");
  PKDA_REQUIRE(a->struct_size == (int32_t)sizeof(*a), PKDA_EINVAL, "pkda_paged_store_args size mismatch");
  StoreParams p;
  if (int st = paged_seqs_from(a, p.s)) return st;
  const int64_t vec = a->dtype == PKDA_BF16 ? 8 : 4;
  const bool fp8 = a->cache_dtype == PKDA_CACHE_FP8;
  PKDA_REQUIRE(fp8 || a->cache_dtype == a->dtype, PKDA_EUNSUPPORTED, "cache_dtype %d", a->cache_dtype);
  if (int st = paged_pointers(a, fp8 ? 16 : vec)) return st;
  if (fp8) {
    if (int st = fp8_head_dim(a->head_dim)) return st;
    if (int st = scale_pointers(a)) return st;
  }
  PKDA_REQUIRE(a->q_heads >= 0 && a->q_heads <= 65535, PKDA_EINVAL, "q_heads %d", a->q_heads);
  PKDA_REQUIRE((a->cos == nullptr) == (a->sin == nullptr), PKDA_EINVAL, "cos without sin");
  const int rotary = a->cos ? a->rotary_dim : 0;
  PKDA_REQUIRE(rotary >= 0 && rotary <= a->head_dim && rotary % 16 == 0, PKDA_EUNSUPPORTED,
               "rotary_dim %d (a multiple of 16 up to head_dim %d)", rotary, a->head_dim);
  PKDA_REQUIRE(rotary == 0 || a->rope_rows >= (int64_t)a->max_pages * a->page_size, PKDA_EINVAL,
               "cos / sin hold %lld positions, a table row %lld", (long long)a->rope_rows,
               (long long)a->max_pages * a->page_size);
  PKDA_REQUIRE(!(a->q_norm || a->k_norm) || a->norm_dtype == PKDA_F32 || a->norm_dtype == PKDA_BF16, PKDA_EUNSUPPORTED,
               "norm_dtype %d", a->norm_dtype);
  if (a->num_tokens == 0) return 0;
  PKDA_REQUIRE(a->k && a->v && (a->q_heads == 0 || (a->q && a->q_out)), PKDA_EINVAL, "null tensor");
  PKDA_REQUIRE((a->k_stride | a->v_stride | (a->q_heads ? a->q_stride : 0)) % vec == 0 &&
                   ((uintptr_t)a->k | (uintptr_t)a->v | (uintptr_t)a->q | (uintptr_t)a->q_out | (uintptr_t)a->cos |
                    (uintptr_t)a->sin | (uintptr_t)a->q_norm | (uintptr_t)a->k_norm) % 16 == 0,
               PKDA_EINVAL, "q, k, v, cos, sin, the norms' weights must be 16-byte aligned");
  p.q = a->q; p.k = a->k; p.v = a->v;
  p.q_stride = a->q_stride; p.k_stride = a->k_stride; p.v_stride = a->v_stride;
  p.q_out = a->q_out; p.k_pages = a->k_pages; p.v_pages = a->v_pages;
  p.k_page_stride = a->k_page_stride; p.v_page_stride = a->v_page_stride;
  p.cos = a->cos; p.sin = a->sin; p.q_heads = a->q_heads; p.kv_heads = a->kv_heads;
  p.rotary = rotary; p.interleaved = a->interleaved;
  p.q_norm = a->q_norm; p.k_norm = a->k_norm; p.norm_bf16 = a->norm_dtype == PKDA_BF16; p.eps = a->eps;
  p.k_scales = a->k_scales; p.v_scales = a->v_scales;
  p.k_scale_stride = a->k_scale_stride; p.v_scale_stride = a->v_scale_stride;
  hipStream_t s = static_cast<hipStream_t>(stream);
  return a->dtype == PKDA_BF16 ? store_dim<bf16_t>(p, a->head_dim, fp8, s) : store_dim<float>(p, a->head_dim, fp8, s);
}
