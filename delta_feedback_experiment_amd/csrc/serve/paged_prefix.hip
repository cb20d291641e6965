// Attention of a batch in groups of sequences that share their first positions
// (gfx950), over a paged cache of the activations' type or of 8-bit floats.
//
// A softmax over two sets of keys is joined from its parts: with each part's
// maximum m_i, sum l_i and weighted values O_i,
//   m = max m_i,  o = sum 2^(m_i - m) O_i / sum 2^(m_i - m) l_i.
// So the rows of a whole group (its sequences' new tokens times the query heads
// of a key/value head) are tiles over the shared positions, which are then read
// once for all of them, and each sequence's rows run over its own positions as in
// plain attention; both in one launch, by the forms of paged_attention.h, every
// part's m, l and O to a workspace in FP32, joined by a second kernel.  The shared
// part takes whole tiles of keys; what is left of a prefix belongs to the
// sequences' own part, so that no tile of keys lies on both sides.
//
// A row whose position lies inside its group's prefix sees what is before it, as
// it would without the group.
#include "paged_attention.h"

namespace pkda {
namespace {

struct PrefixPlan {
  Plan shared, own;
};

// The two parts' forms and splits, from what the host knows.
inline PrefixPlan prefix_plan(AttnParams& shared, AttnParams& own) {
  PrefixPlan r;
  AttnParams groups = shared;  // to the rules a group is a sequence
  groups.s.num_seqs = shared.num_groups;
  r.shared = plan(groups, true);
  shared.splits = groups.splits < kMaxSplits / 2 ? groups.splits : kMaxSplits / 2;
  shared.min_chunk = groups.min_chunk;
  shared.key_rows = groups.key_rows;
  shared.whole = 0;
  if (groups.key_rows == 32) r.shared.key_tiles = shared.num_groups;
  r.own = plan(own, own.s.cu != nullptr);
  if (own.splits > kMaxSplits / 2) own.splits = kMaxSplits / 2;
  return r;
}

template <typename G>
int launch_prefix(AttnParams shared, AttnParams own, hipStream_t s) {
  constexpr const char* what = "pkda_paged_prefix_attention";
  const PrefixPlan r = prefix_plan(shared, own);
  const int64_t shared_tile = (int64_t)shared.kv_heads * shared.splits, own_tile = (int64_t)own.kv_heads * own.splits;
  const int64_t first = (r.shared.row_tiles + r.shared.key_tiles) * shared_tile;
  const int64_t blocks = first + (r.own.row_tiles + r.own.key_tiles) * own_tile;
  const int64_t rows = (int64_t)own.s.num_tokens * own.q_heads;
  PKDA_REQUIRE(blocks <= INT32_MAX && rows <= INT32_MAX, PKDA_EINVAL, "%d tokens of %d heads", own.s.num_tokens,
               own.q_heads);
  shared.row_blocks = (unsigned)(r.shared.row_tiles * shared_tile);
  own.row_blocks = (unsigned)(r.own.row_tiles * own_tile);
  // the parts of a row: the shared ones, then its own
  own.part_o = shared.part_o + shared.splits * rows * G::D;
  own.part_ml = shared.part_ml + shared.splits * rows * 2;
  const dim3 grid((unsigned)blocks), block(kThreads);
  if (own.s.page_size % (64 / G::SC) == 0)
    hipLaunchKernelGGL((paged_prefix_kernel<G, true>), grid, block, 0, s, shared, own, (unsigned)first);
  else
    hipLaunchKernelGGL((paged_prefix_kernel<G, false>), grid, block, 0, s, shared, own, (unsigned)first);
  if (int st = launch_status(what)) return st;
  return launch_join<G, true>(shared, own, s, what);
}

template <typename T>
int prefix_dim(const AttnParams& shared, const AttnParams& own, int dim, bool fp8, hipStream_t s) {
  if (fp8)
    return dim == 128 ? launch_prefix<Geo<T, 128, true>>(shared, own, s) : launch_prefix<Geo<T, 64, true>>(shared, own, s);
  return dim == 128  ? launch_prefix<Geo<T, 128, false>>(shared, own, s)
         : dim == 64 ? launch_prefix<Geo<T, 64, false>>(shared, own, s)
                     : launch_prefix<Geo<T, 32, false>>(shared, own, s);
}

int sizes_of(const pkda_paged_prefix_args* a, AttnParams& p) {
  PKDA_REQUIRE(a != nullptr, PKDA_EINVAL, "null args");
  PKDA_REQUIRE(a->struct_size == (int32_t)sizeof(*a), PKDA_EINVAL, "pkda_paged_prefix_args size mismatch");
  if (int st = attention_sizes(a, p)) return st;
  PKDA_REQUIRE(a->num_groups >= 0 && a->num_groups <= 1 << 30, PKDA_EINVAL, "num_groups %d", a->num_groups);
  p.num_groups = a->num_groups;
  return 0;
}

}  // namespace
}  // namespace pkda

extern "C" int64_t pkda_paged_prefix_workspace(const pkda_paged_prefix_args* a) {
  using namespace pkda;
  AttnParams shared;
  if (sizes_of(a, shared)) return -1;
  // by the sizes alone: one token a sequence may come with cu_seqlens or without
  int splits = 0;
  for (const bool packed : {true, false}) {
    if (!packed && a->num_tokens != a->num_seqs) continue;
    AttnParams own = shared, both = shared;
    own.s.cu = both.s.cu = packed ? reinterpret_cast<const int32_t*>(16) : nullptr;  // whether, not where
    prefix_plan(both, own);
    splits = splits > both.splits + own.splits ? splits : both.splits + own.splits;
  }
  return (int64_t)splits * a->num_tokens * a->q_heads * (a->head_dim + 2);
}

extern "C" int pkda_paged_prefix_attention(const pkda_paged_prefix_args* a, void* stream) {
  using namespace pkda;
  AttnParams shared;
  if (int st = sizes_of(a, shared)) return st;
  const bool fp8 = a->k_scales || a->v_scales;
  const int64_t vec = a->dtype == PKDA_BF16 ? 8 : 4;
  if (int st = paged_pointers(a, fp8 ? 16 : vec)) return st;
  if (fp8) {
    if (int st = fp8_head_dim(a->head_dim)) return st;
    if (int st = scale_pointers(a)) return st;
  }
  PKDA_REQUIRE(a->num_groups == 0 || (a->cu_groups && a->prefix_lens), PKDA_EINVAL, "null groups");
  if (a->num_tokens == 0) return 0;
  AttnParams own = shared;
  prefix_plan(shared, own);
  if (int st = attention_tensors(a, shared, vec, shared.splits + own.splits)) return st;
  PKDA_REQUIRE(shared.part_o, PKDA_EINVAL, "workspace");
  shared.k_scales = a->k_scales; shared.v_scales = a->v_scales;
  shared.k_scale_stride = a->k_scale_stride; shared.v_scale_stride = a->v_scale_stride;
  shared.groups = a->cu_groups; shared.prefix_lens = a->prefix_lens;
  own = shared;
  hipStream_t s = static_cast<hipStream_t>(stream);
  return a->dtype == PKDA_BF16 ? prefix_dim<bf16_t>(shared, own, a->head_dim, fp8, s)
                               : prefix_dim<float>(shared, own, a->head_dim, fp8, s);
}
