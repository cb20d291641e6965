// Attention of new tokens over a paged cache of 8-bit floats (gfx950): the forms
// of paged_attention.h, whose loads take a row's codes, half the bytes of BF16,
// and its scales, a byte for each 32 channels.
//
// Codes become operands of the queries' type on their way to the products: the
// conversion multiplies by the block's scale, a power of two, so that it is exact
// and nothing is rounded but what the same attention over a BF16 cache rounds.
// Up to 32 rows a sequence a lane converts its key's chunks in registers, the
// keys' for the first product and the values' on their way to LDS; more rows
// convert what they stage, so that a number is converted once for 128 rows.
//
// What bounds it, in BF16 with heads of 128 (a 4 GiB copy runs at 4.55 TB/s).
// Decode, 256 sequences of 325 to 4,875 keys, 32/8 heads: 288 us, 4.95 TB/s of codes
// and scales (547 us over a BF16 cache).  4 sequences of 700 keys: 5.9 us and 3.6 for
// the join, a trip to memory after the other.  2,048 tokens after 14,336: 598 to 626 us
// by box, 823 to 861 TFLOP/s, what the same takes over a BF16 cache: softmax beside
// products.  Several new tokens, or one with cu_seqlens, run in the 32-row form in the
// caller's order: those 256 sequences with one token so 349 us (4.2 TB/s), with five
// 370 (3.9; 630 over a BF16 cache); 64 of them with five 124 (3.0; 192).  FP32 queries:
// 465 us with one token, 1,228 where that comes with cu_seqlens, 1,266 with five.
#include "paged_attention.h"

namespace pkda {
namespace {

template <typename T>
int attention_fp8_dim(const AttnParams& p, int dim, hipStream_t s) {
  constexpr const char* what = "pkda_paged_attention_fp8";
  return dim == 128 ? launch_attention<Geo<T, 128, true>>(p, s, what) : launch_attention<Geo<T, 64, true>>(p, s, what);
}

int sizes_of(const pkda_paged_attention_fp8_args* a, AttnParams& p) {
  PKDA_REQUIRE(a != nullptr, PKDA_EINVAL, "null args");
  PKDA_REQUIRE(a->struct_size == (int32_t)sizeof(*a), PKDA_EINVAL, "pkda_paged_attention_fp8_args size mismatch");
  if (int st = attention_sizes(a, p)) return st;
  return fp8_head_dim(a->head_dim);
}

}  // namespace
}  // namespace pkda

extern "C" int64_t pkda_paged_attention_fp8_workspace(const pkda_paged_attention_fp8_args* a) {
  pkda::AttnParams p;
  if (pkda::sizes_of(a, p)) return -1;
  return pkda::attention_workspace(a, p);
}

extern "C" int pkda_paged_attention_fp8(const pkda_paged_attention_fp8_args* a, void* stream) {
  using namespace pkda;
  AttnParams p;
  if (int st = sizes_of(a, p)) return st;
  if (int st = paged_pointers(a, 16)) return st;
  if (int st = scale_pointers(a)) return st;
  if (a->num_tokens == 0) return 0;
  if (int st = attention_tensors(a, p, a->dtype == PKDA_BF16 ? 8 : 4, p.splits)) return st;
  p.k_scales = a->k_scales; p.v_scales = a->v_scales;
  p.k_scale_stride = a->k_scale_stride; p.v_scale_stride = a->v_scale_stride;
  hipStream_t s = static_cast<hipStream_t>(stream);
  return a->dtype == PKDA_BF16 ? attention_fp8_dim<bf16_t>(p, a->head_dim, s) : attention_fp8_dim<float>(p, a->head_dim, s);
}
