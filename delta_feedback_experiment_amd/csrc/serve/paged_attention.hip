// Attention of new tokens over a paged key/value cache of the activations' type
// (gfx950): the forms of paged_attention.h, which says what they compute and what
// bounds them.
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
