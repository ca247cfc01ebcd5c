// Attention of rows at any positions over dense keys (CacheBlend's recomputed
// rows, packed documents): a pass over the keys' positions, the tensor-core
// kernel, and a join when the keys are split.
#include <algorithm>

#include "split_attention.cuh"
#include "tensor_maps.h"

namespace lmc {
namespace {

// Positions as 32-bit integers padded to whole tiles with one that no row sees,
// and each tile's range, so that a block can skip tiles or leave out the masks.
__global__ void __launch_bounds__(kTileN)
    key_tiles_kernel(PositionArgs a, int *pos32, int *doc32, float *rel, TileStats *stats,
                     int *run) {
  __shared__ int edge[4][4], first;
  let_next_start();
  const int tile = blockIdx.x, i = tile * kTileN + threadIdx.x;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr int kLow = -2147483647 - 1, kHigh = 2147483647;
  const bool in = i < a.k_tokens;
  const int p = !in ? kHigh : a.k_pos ? clamp_pos(position_at(a.k_pos, a.long_k_pos, i)) : i;
  const int d = in && a.k_doc ? a.k_doc[i] : in ? 0 : -1;
  int lo = __reduce_min_sync(0xffffffffu, p), hi = __reduce_max_sync(0xffffffffu, p);
  int d_lo = __reduce_min_sync(0xffffffffu, in ? d : kHigh);
  int d_hi = __reduce_max_sync(0xffffffffu, in ? d : kLow);
  if (lane == 0) edge[0][warp] = lo, edge[1][warp] = hi, edge[2][warp] = d_lo, edge[3][warp] = d_hi;
  if (threadIdx.x == 0) first = p;
  __syncthreads();
  const bool one_apart =
      __syncthreads_and(!in || p - static_cast<long long>(first) == threadIdx.x);
  lo = min(min(edge[0][0], edge[0][1]), min(edge[0][2], edge[0][3]));
  pos32[i] = p;
  doc32[i] = d;
  rel[i] = static_cast<float>(static_cast<long long>(p) - lo);
  if (threadIdx.x == 0) {
    hi = max(max(edge[1][0], edge[1][1]), max(edge[1][2], edge[1][3]));
    d_lo = min(min(edge[2][0], edge[2][1]), min(edge[2][2], edge[2][3]));
    d_hi = max(max(edge[3][0], edge[3][1]), max(edge[3][2], edge[3][3]));
    stats[tile] = {lo, hi, d_lo, d_hi};
    run[tile] = one_apart;
  }
}

struct Plan {
  bool split;  // the kernel for few rows or keys; else the tensor-core kernel
  int row_tiles;
  int tiles, per_slice, slices, groups;  // slices == 0: not split
  long long keys;                        // padded
};

// Blocks of 16 rows times steps of 64 keys up to which the split kernel is taken.
// Measured (B200, 32/8 heads, split / tensor cores, us, replayed without host calls):
//                         steps  D 128        D 64         D 128, cap and bias
//   38 rows on 257 keys     400   9.3 / 15.0   7.1 / 12.0  11.1 / 20.3
//   128 on 512             2048  14.9 / 18.4  10.6 / 15.8  17.7 / 28.2
//   1 on 16384             2048  20.7 / 23.0  14.9 / 20.1  19.9 / 33.6
//   256 on 512             4096  27.9 / 17.6  20.2 / 14.8  32.8 / 27.7
//   8 at the end of 16384  4096  27.2 / 24.5  18.4 / 20.8  32.4 / 36.4
//   8 spread over 16384    4096  28.2 / 48.8  19.5 / 46.7  33.4 / 61.6
// Rows far apart cost the tensor-core kernel its masks (nearly every tile is in part
// visible to a warp's rows), which the sizes do not tell; the border is where rows
// next to one another break even.
constexpr long long kSplitSteps = 2048;

// The keys are split when the blocks would not fill the GPU: towards one block
// per SM, with at least four tiles each (below that the join costs more than
// the shorter stream saves).
Plan plan_of(const PositionArgs &a) {
  Plan p = {};
  p.tiles = (a.k_tokens + kTileN - 1) / kTileN;
  p.keys = static_cast<long long>(p.tiles) * kTileN;
  const long long rows = static_cast<long long>(a.q_tokens) * (a.heads / a.kv_heads);
  p.groups = static_cast<int>((rows + kBlockRows - 1) / kBlockRows);
  p.row_tiles = static_cast<int>((rows + kSplitRows - 1) / kSplitRows);
  const long long steps = static_cast<long long>(p.row_tiles) * a.kv_heads *
                          ((a.k_tokens + kSplitWarps * kSplitKeys - 1) / (kSplitWarps * kSplitKeys));
  if (steps <= kSplitSteps) {
    p.split = true;
    p.slices = split_slices(static_cast<long long>(p.row_tiles) * a.kv_heads, a.k_tokens);
    return p;
  }
  const long long blocks = static_cast<long long>(p.groups) * a.kv_heads;
  const long long want = std::min(148 / std::max(1ll, blocks), p.tiles / 4ll);
  p.slices = want >= 2 ? static_cast<int>(want) : 0;
  p.per_slice = p.slices ? (p.tiles + p.slices - 1) / p.slices : p.tiles;
  if (p.slices) p.slices = (p.tiles + p.per_slice - 1) / p.per_slice;
  return p;
}

template <typename T, int D>
cudaError_t launch(const PositionArgs &a, void *workspace, cudaStream_t stream) {
  const Plan p = plan_of(a);
  const long long rows = static_cast<long long>(a.q_tokens) * a.heads;
  if (p.split) {
    const bool joined = p.slices > kMostClustered;  // else the parts join in a cluster
    float *part_o = joined ? static_cast<float *>(workspace) : nullptr;
    float *part_lse = joined ? part_o + p.slices * rows * D : nullptr;
    const SplitPass s = {0, 0, false, a.q_tokens, p.row_tiles, p.slices,
                         a.heads / a.kv_heads, part_o, part_lse};
    cudaError_t e = launch_split<T, D>(a, s, 1, true, stream);
    if (e != cudaSuccess || !joined) return e;
    return launch_ordered(join_position_kernel<T, D>, dim3(static_cast<unsigned>((rows + 3) / 4)),
                          128, 0, false, stream, 1, a, part_o, part_lse, p.slices);
  }
  char *w = static_cast<char *>(workspace);
  TileStats *stats = reinterpret_cast<TileStats *>(w);
  w += p.tiles * sizeof(TileStats);
  int *pos32 = reinterpret_cast<int *>(w);
  int *doc32 = pos32 + p.keys;
  float *rel = reinterpret_cast<float *>(doc32 + p.keys);
  int *run = reinterpret_cast<int *>(rel + p.keys);
  w = reinterpret_cast<char *>(run + (p.tiles + 3) / 4 * 4);
  TcArgs t = {};
  t.part_o = reinterpret_cast<float *>(w);
  t.part_lse = t.part_o + p.slices * rows * D;
  key_tiles_kernel<<<p.tiles, kTileN, 0, stream>>>(a, pos32, doc32, rel, stats, run);
  t.q = a.q, t.out = a.out, t.lse = a.lse, t.slopes = a.slopes;
  t.q_batch = 0, t.q_token = a.q_token, t.q_head = a.q_head;
  t.tokens = t.q_len = a.q_tokens;
  t.heads = a.heads, t.group = a.heads / a.kv_heads;
  t.k_tiles = p.tiles, t.tiles_per_slice = p.per_slice, t.slices = p.slices;
  set_scores(t, a.scale, a.softcap);
  t.pos = a;
  t.k_pos32 = pos32, t.k_doc32 = a.k_doc ? doc32 : nullptr, t.k_rel = rel, t.stats = stats;
  t.k_run = run;
  CUtensorMap k_map, v_map;
  const long long dims[3] = {D, a.kv_heads, a.k_tokens};
  const long long ks[2] = {a.k_head, a.k_token}, vs[2] = {a.v_head, a.v_token};
  const int box[3] = {64, 1, kTileN};
  constexpr bool kBf16 = __is_same(T, __nv_bfloat16);
  if (!encode_rows(&k_map, kBf16, a.k, 3, dims, ks, box) ||
      !encode_rows(&v_map, kBf16, a.v, 3, dims, vs, box))
    return cudaErrorInvalidValue;
  const unsigned grid = static_cast<unsigned>(p.groups) * a.kv_heads * std::max(1, p.slices);
  cudaError_t e = t.k_doc32 ? launch_tc<T, D, true, true>(k_map, v_map, t, grid, false, stream)
                            : launch_tc<T, D, true, false>(k_map, v_map, t, grid, false, stream);
  if (e != cudaSuccess || !p.slices) return e;
  return launch_ordered(join_position_kernel<T, D>, dim3(static_cast<unsigned>((rows + 3) / 4)), 128,
                        0, false, stream, 1, a, t.part_o, t.part_lse, p.slices);
}

}  // namespace

PositionPasses position_passes(const PositionArgs &a) {
  const Plan p = plan_of(a);
  if (p.split) return {0, p.slices};
  return {std::max(1, p.slices), 0};
}

long long position_attention_workspace(const PositionArgs &a, int dim) {
  const Plan p = plan_of(a);
  if (p.split)
    return p.slices <= kMostClustered
               ? 0
               : p.slices * static_cast<long long>(a.q_tokens) * a.heads * (dim + 1) * 4;
  return p.tiles * static_cast<long long>(sizeof(TileStats)) + p.keys * 12 + (p.tiles + 3) / 4 * 16 +
         p.slices * static_cast<long long>(a.q_tokens) * a.heads * (dim + 1) * 4;
}

cudaError_t launch_position_attention(const PositionArgs &a, RowType type, int dim,
                                      void *workspace, cudaStream_t stream) {
  if (type == RowType::kBFloat16)
    return dim == 64 ? launch<__nv_bfloat16, 64>(a, workspace, stream)
                     : launch<__nv_bfloat16, 128>(a, workspace, stream);
  return dim == 64 ? launch<__half, 64>(a, workspace, stream)
                   : launch<__half, 128>(a, workspace, stream);
}

}  // namespace lmc
