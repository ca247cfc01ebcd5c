// Attention of a batch over a shared prefix in pages: one warp per row, by the
// definition.
#include <algorithm>

#include "attention.cuh"

namespace lmc {
namespace {

template <typename T, int D>
__global__ void __launch_bounds__(128) paged_rows_kernel(PagedArgs a) {
  const long long rows = static_cast<long long>(a.batch) * a.q_len * a.heads;
  const int group = a.heads / a.kv_heads;
  for (long long r = static_cast<long long>(blockIdx.x) * 4 + (threadIdx.x >> 5); r < rows;
       r += static_cast<long long>(gridDim.x) * 4) {
    const int h = static_cast<int>(r % a.heads);
    const int i = static_cast<int>(r / a.heads % a.q_len);
    const int b = static_cast<int>(r / a.heads / a.q_len);
    const int n = max(0, a.own_lens[b]);
    const long long pos = a.prefix_len + n - a.q_len + i;
    const long long own = max(0ll, static_cast<long long>(n) - a.q_len + i + 1);
    const float slope = a.slopes ? a.slopes[h] : 0.f;
    WarpRow<T, D> row;
    row.start(static_cast<const T *>(a.q) + b * a.q_batch + i * a.q_token + h * a.q_head);
    for (long long j = 0; j < a.prefix_len + own; ++j) {
      const bool shared = j < a.prefix_len;
      const long long at = shared ? j : j - a.prefix_len;
      const long long col = at / a.block_size, off = at - col * a.block_size;
      if (!shared && col >= a.width) {
        if ((threadIdx.x & 31) == 0) report_status(a.status, kStatusBadIndex, b, n, a.width);
        break;
      }
      const int page = shared ? a.prefix_blocks[col] : a.tables[b * a.table_stride + col];
      if (page < 0 || page >= a.num_blocks) {
        if ((threadIdx.x & 31) == 0) report_status(a.status, kStatusBadSlot, b, col, page);
        continue;
      }
      const float gap = fabsf(static_cast<float>(pos - j));
      row.add(static_cast<const T *>(a.k) + page * a.k_block + off * a.k_slot +
                  h / group * a.k_head,
              static_cast<const T *>(a.v) + page * a.v_block + off * a.v_slot +
                  h / group * a.v_head,
              a.scale, a.softcap, slope * gap);
    }
    row.finish(static_cast<T *>(a.out) + r * D, a.lse ? a.lse + r : nullptr);
  }
}

}  // namespace

cudaError_t launch_shared_prefix_attention(const PagedArgs &a, RowType type, int dim,
                                           cudaStream_t stream) {
  const long long rows = static_cast<long long>(a.batch) * a.q_len * a.heads;
  const unsigned grid = static_cast<unsigned>(std::min((rows + 3) / 4, 1ll << 20));
#define LMC_ROWS(T, D) paged_rows_kernel<T, D><<<grid, 128, 0, stream>>>(a)
  if (type == RowType::kBFloat16) {
    if (dim == 64) LMC_ROWS(__nv_bfloat16, 64); else LMC_ROWS(__nv_bfloat16, 128);
  } else {
    if (dim == 64) LMC_ROWS(__half, 64); else LMC_ROWS(__half, 128);
  }
#undef LMC_ROWS
  return cudaGetLastError();
}

}  // namespace lmc
