// Attention of a batch over a prefix that its requests share: the prefix in
// whole 128-key tiles once for all rows on the tensor cores, the rest of the
// prefix and each request's own keys in a pass that is split over the keys, and
// a join of the parts.
#include <algorithm>

#include "split_attention.cuh"
#include "tensor_maps.h"

namespace lmc {
namespace {

struct PrefixPlan {
  int tiles, per_slice, tc_slices, groups;  // tensor-core pass over tiles * 128 keys
  int pre_slices, pre_tiles;                // split pass of all rows over the prefix
  int own_begin, own_slices, own_tiles;     // split pass per request, from this prefix key on
};

// Blocks of 16 rows times steps of 64 keys up to which the split pass reads the
// prefix.  Measured (B200, 32/8 heads, split / tensor cores, us, replayed without
// host calls):          steps  D 128        D 64         D 128, cap and bias
//   8 requests on 4096   1024  17.9 / 19.6  16.0 / 17.9  20.0 / 24.1
//   1 on 16000           2000  21.7 / 24.6  20.6 / 22.1  24.8 / 32.1
//   64 on 1024           2048  23.9 / 22.2  17.8 / 18.2  28.8 / 27.3
//   32 on 4096           4096  29.2 / 21.5  21.1 / 18.9  36.4 / 25.6
constexpr long long kSplitSteps = 2000;
// ... and up to which every request reads it with its own keys, in one pass and one
// launch instead of two and three (one / two passes: 4 on 500 tokens, 256 steps,
// 7.9 / 10.2, D 64 6.4 / 9.0, capped 9.9 / 12.2; 16 on 500, 1024 steps, 11.0 / 11.6,
// 8.0 / 10.1, 12.8 / 13.8; 16 on 1024, 2048 steps, 15.0 / 13.3, 10.6 / 11.6,
// 18.7 / 14.9).
constexpr long long kFewSteps = 1200;

PrefixPlan plan_of(const PagedArgs &a) {
  PrefixPlan p = {};
  const int group = a.heads / a.kv_heads, bs = a.block_size;
  const long long tokens = static_cast<long long>(a.batch) * a.q_len;
  const int prefix = static_cast<int>(a.prefix_len);
  // whole pages or whole 128-slot parts of them must make up a tile, in 8-row
  // groups of the swizzle
  const bool boxes = bs % 8 == 0 && (kTileN % bs == 0 || bs % kTileN == 0);
  const long long row_tiles = (tokens * group + kSplitRows - 1) / kSplitRows;
  const long long prefix_steps = (prefix + kSplitWarps * kSplitKeys - 1) / (kSplitWarps * kSplitKeys);
  const long long request_tiles = (a.q_len * group + kSplitRows - 1) / kSplitRows;
  if (a.batch * request_tiles * a.kv_heads * prefix_steps <= kFewSteps) {
    // one pass
  } else if (boxes && prefix >= kTileN && row_tiles * a.kv_heads * prefix_steps > kSplitSteps) {
    p.tiles = prefix / kTileN;
    p.groups = static_cast<int>((tokens * group + kBlockRows - 1) / kBlockRows);
    const long long blocks = static_cast<long long>(p.groups) * a.kv_heads;
    const long long want = std::max(1ll, std::min({148 / blocks, p.tiles / 2ll, 64ll}));
    p.per_slice = static_cast<int>((p.tiles + want - 1) / want);
    p.tc_slices = (p.tiles + p.per_slice - 1) / p.per_slice;
    p.own_begin = p.tiles * kTileN;
  } else if (a.batch > 1) {
    p.pre_tiles = static_cast<int>(row_tiles);
    p.pre_slices = split_slices(row_tiles * a.kv_heads, prefix);
    p.own_begin = prefix;
  }
  p.own_tiles = (a.q_len * group + kSplitRows - 1) / kSplitRows;
  p.own_slices =
      split_slices(static_cast<long long>(a.batch) * p.own_tiles * a.kv_heads,
                   prefix - p.own_begin + static_cast<long long>(a.width) * a.block_size);
  return p;
}

// One pass of few parts per row needs no workspace: they join in a cluster.
bool needs_join(const PrefixPlan &p) {
  return p.tc_slices + p.pre_slices > 0 || p.own_slices > kMostClustered;
}

template <typename T, int D>
cudaError_t launch(const PagedArgs &a, void *workspace, cudaStream_t stream) {
  const PrefixPlan p = plan_of(a);
  const long long rows = static_cast<long long>(a.batch) * a.q_len * a.heads;
  const int slices = p.tc_slices + p.pre_slices + p.own_slices, group = a.heads / a.kv_heads;
  const bool joined = needs_join(p);
  float *part_o = static_cast<float *>(workspace);
  float *part_lse = part_o + slices * rows * D;
  cudaError_t e = cudaSuccess;
  if (p.tc_slices) {
    TcArgs t = {};
    t.q = a.q, t.slopes = a.slopes;
    t.q_batch = a.q_batch, t.q_token = a.q_token, t.q_head = a.q_head;
    t.tokens = a.batch * a.q_len, t.q_len = a.q_len;
    t.heads = a.heads, t.group = a.heads / a.kv_heads;
    t.k_tiles = p.tiles, t.tiles_per_slice = p.per_slice, t.slices = p.tc_slices;
    t.part_o = part_o, t.part_lse = part_lse;
    set_scores(t, a.scale, a.softcap);
    t.pages = a.prefix_blocks, t.own_lens = a.own_lens;
    t.block_size = a.block_size, t.num_blocks = a.num_blocks, t.prefix_len = a.prefix_len;
    t.status = a.status;
    CUtensorMap k_map, v_map;
    const long long dims[4] = {D, a.kv_heads, a.block_size, a.num_blocks};
    const long long ks[3] = {a.k_head, a.k_slot, a.k_block};
    const long long vs[3] = {a.v_head, a.v_slot, a.v_block};
    const int box[4] = {64, 1, std::min(kTileN, a.block_size), 1};
    constexpr bool kBf16 = __is_same(T, __nv_bfloat16);
    if (!encode_rows(&k_map, kBf16, a.k, 4, dims, ks, box) ||
        !encode_rows(&v_map, kBf16, a.v, 4, dims, vs, box))
      return cudaErrorInvalidValue;
    const unsigned grid = static_cast<unsigned>(p.groups) * a.kv_heads * p.tc_slices;
    e = launch_tc<T, D, false, false>(k_map, v_map, t, grid, true, stream);
    if (e != cudaSuccess) return e;
  }
  int first = p.tc_slices;
  if (p.pre_slices) {
    const SplitPass s = {0, static_cast<int>(a.prefix_len), false, a.batch * a.q_len, p.pre_tiles,
                         p.pre_slices, group, part_o + first * rows * D, part_lse + first * rows};
    e = launch_split<T, D>(a, s, 1, true, stream);
    if (e != cudaSuccess) return e;
    first += p.pre_slices;
  }
  const SplitPass s = {p.own_begin, static_cast<int>(a.prefix_len), true, a.q_len, p.own_tiles,
                       p.own_slices, group, joined ? part_o + first * rows * D : nullptr,
                       part_lse + first * rows};
  e = launch_split<T, D>(a, s, a.batch, first == 0, stream);
  if (e != cudaSuccess || !joined) return e;
  return launch_ordered(join_paged_kernel<T, D>, dim3(static_cast<unsigned>((rows + 3) / 4)), 128, 0,
                        false, stream, 1, a, part_o, part_lse, slices);
}

}  // namespace

PrefixPasses prefix_passes(const PagedArgs &a) {
  const PrefixPlan p = plan_of(a);
  return {p.tc_slices, p.pre_slices, p.own_slices};
}

long long shared_prefix_attention_workspace(const PagedArgs &a, int dim) {
  const PrefixPlan p = plan_of(a);
  const int slices = p.tc_slices + p.pre_slices + p.own_slices;
  return !needs_join(p) ? 0
                     : static_cast<long long>(slices) * a.batch * a.q_len * a.heads * (dim + 1) * 4;
}

cudaError_t launch_shared_prefix_attention(const PagedArgs &a, RowType type, int dim,
                                           void *workspace, cudaStream_t stream) {
  if (type == RowType::kBFloat16)
    return dim == 64 ? launch<__nv_bfloat16, 64>(a, workspace, stream)
                     : launch<__nv_bfloat16, 128>(a, workspace, stream);
  return dim == 64 ? launch<__half, 64>(a, workspace, stream)
                   : launch<__half, 128>(a, workspace, stream);
}

}  // namespace lmc
