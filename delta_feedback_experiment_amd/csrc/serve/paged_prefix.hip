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
// Which of a group's pages the shared positions are read from is this file's to
// choose, since all of the sequences that hold them hold the same there: the first
// such sequence's, which a wave finds by 64 lengths at a time (under 1 us of a
// tile's way to its keys).
//
// A row whose position lies inside its group's prefix sees what is before it, as
// it would without the group.
//
// Parts are taken whatever the numbers of new tokens, which the host does not know a
// sequence at a time: by their mean one long chunk would decide for the sequences that
// decode beside it.  Those are what parts are for (32/8 heads, us by parts and each
// sequence whole: 60 of one token and one of 1,920 behind 16,384 682 and 1,037, one of
// 3,900 1,398 and 1,742; 250 and one of 8,192 behind 8,192 2,118 and 2,750).  Long
// chunks alone are better off whole, which their caller can have from the plain
// attention (16 sequences behind 4,096, 33 tokens each 146 and 131, 96 tokens 198 and
// 168, 512 tokens 874 and 689: two parts of a row are 2 x 1 KB of FP32 a head).
#include "paged_attention.h"

namespace pkda {
namespace {

struct PrefixPlan {
  Plan shared, own;
};

// The two parts' forms and splits, from what the host knows.
inline PrefixPlan prefix_plan(AttnParams& shared, AttnParams& own) {
  PrefixPlan r;
  const int64_t group = shared.group.d, N = shared.s.num_tokens, G = shared.num_groups, heads = shared.kv_heads;
  // Groups of more than 32 rows are tiles of 128, however few: their keys are split
  // over one workgroup a compute unit, so that the own parts' workgroups, which wait
  // for memory, run beside them.  64 sequences of 300 keys behind 16,384, 32/8 heads:
  // 57 us with splits for 256 workgroups, 60 with 384, 64 with 512 (and 103 where the
  // own part has four splits); of at least 256 keys, which 32 sequences of 5 tokens
  // behind 7,000 take 34 us with, 512 keys 34, 1,024 37, 6 groups of 16 behind 2,500
  // 28, 30 and 42.
  shared.key_rows = 32;
  r.shared.row_tiles = tile_bound(N, G, group, kRowTile, true);
  r.shared.key_tiles = G;
  const int64_t per_group = G > 0 ? (N * group + G - 1) / G : 0;
  const int64_t tiles = per_group > 32 ? G * ((per_group + kRowTile - 1) / kRowTile) : G;
  shared.min_chunk = per_group > 32 ? 256 : kMinChunk;
  int64_t want = kSlots / 2 / (tiles * heads > 0 ? tiles * heads : 1);
  const int64_t cap = ((int64_t)shared.s.max_pages * shared.s.page_size + shared.min_chunk - 1) / shared.min_chunk;
  if (want > cap) want = cap;
  if (want > kMaxSplits / 2) want = kMaxSplits / 2;
  shared.splits = want < 1 ? 1 : (int)want;
  shared.whole = 0;
  r.own = plan(own, own.s.cu != nullptr);
  // What the sequences hold by themselves is not known here, and seldom long: no more
  // workgroups than the card holds.  The same 64 sequences take 57 us, with four times
  // as many 76, the 6 groups 28 and 32; 8 sequences of 3,000 behind 2,048 31 and 37.
  const int64_t items = (r.own.row_tiles + r.own.key_tiles) * heads;
  int64_t most = kSlots / (items > 0 ? items : 1);
  most = most < 1 ? 1 : most < kMaxSplits / 2 ? most : kMaxSplits / 2;
  if (own.splits > most) own.splits = (int)most;
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
  const bool few = !own.s.cu && own.group.d <= kFewRows, whole = own.s.page_size % (64 / G::SC) == 0;
  const auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, s, shared, own, (unsigned)first); };
  if (few && whole) launch(paged_prefix_kernel<G, true, true>);
  else if (few) launch(paged_prefix_kernel<G, false, true>);
  else if (whole) launch(paged_prefix_kernel<G, true, false>);
  else launch(paged_prefix_kernel<G, false, false>);
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
  shared.k_scales = a->k_scales; shared.v_scales = a->v_scales;
  shared.k_scale_stride = a->k_scale_stride; shared.v_scale_stride = a->v_scale_stride;
  shared.groups = a->cu_groups; shared.prefix_lens = a->prefix_lens;
  own = shared;
  hipStream_t s = static_cast<hipStream_t>(stream);
  return a->dtype == PKDA_BF16 ? prefix_dim<bf16_t>(shared, own, a->head_dim, fp8, s)
                               : prefix_dim<float>(shared, own, a->head_dim, fp8, s);
}
