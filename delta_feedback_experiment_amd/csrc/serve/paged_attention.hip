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
#include "paged_attention.h"

namespace pkda {
namespace {

template <typename T>
int attention_dim(const AttnParams& p, int dim, hipStream_t s) {
  constexpr const char* what = "pkda_paged_attention";
  return dim == 128  ? launch_attention<Geo<T, 128, false>>(p, s, what)
         : dim == 64 ? launch_attention<Geo<T, 64, false>>(p, s, what)
                     : launch_attention<Geo<T, 32, false>>(p, s, what);
}

int sizes_of(const pkda_paged_attention_args* a, AttnParams& p) {
  PKDA_REQUIRE(a != nullptr, PKDA_EINVAL, "null args");
  PKDA_REQUIRE(a->struct_size == (int32_t)sizeof(*a), PKDA_EINVAL, "pkda_paged_attention_args size mismatch");
  return attention_sizes(a, p);
}

}  // namespace
}  // namespace pkda

extern "C" int64_t pkda_paged_attention_workspace(const pkda_paged_attention_args* a) {
  pkda::AttnParams p;
  if (pkda::sizes_of(a, p)) return -1;
  return pkda::attention_workspace(a, p);
}

extern "C" int pkda_paged_attention(const pkda_paged_attention_args* a, void* stream) {
  using namespace pkda;
  AttnParams p;
  if (int st = sizes_of(a, p)) return st;
  const int64_t vec = a->dtype == PKDA_BF16 ? 8 : 4;
  if (int st = paged_pointers(a, vec)) return st;
  if (a->num_tokens == 0) return 0;
  if (int st = attention_tensors(a, p, vec, p.splits)) return st;
  hipStream_t s = static_cast<hipStream_t>(stream);
  return a->dtype == PKDA_BF16 ? attention_dim<bf16_t>(p, a->head_dim, s) : attention_dim<float>(p, a->head_dim, s);
}
