// Arguments of the serving operators' kernels (slot maps, rotary with cache
// writes, attention), without torch: the launchers' checks are in
// serving_ops.cpp, so a kernel file compiles in seconds.
#pragma once
#include <cuda_runtime.h>

#include <cmath>

namespace lmc {

struct DeviceStatus;                 // common.cuh
constexpr int kDeviceStatusBytes = 24;

// Base-2 log of a row's sum from its maximum m and the sum l of its weights; -inf
// for a row without keys.  Such a part is left out of a join, so a row whose wait
// ran out (`whole` false) must not have it even where l is still 0, nor one whose
// scores are all -inf (it has weights, but no maximum): their log is NaN, and the
// join computes the row again.
__host__ __device__ inline float log2_of_sum(bool whole, float m, float l) {
  if (!whole || (l != 0.f && m == -INFINITY)) return NAN;
  return l == 0.f ? -INFINITY : m + log2f(l);
}

enum class RowType { kFloat, kBFloat16, kHalf };

// Slot maps: request lengths in, slots, positions and grown tables out.
struct SlotArgs {
  const void *ctx, *fresh;  // int32 or int64 [B]
  int *tables;              // [B, width], row stride table_stride
  const int *free_blocks;   // [num_free], read when `grow`
  bool grow;                // take missing pages from free_blocks
  long long table_stride, num_free, num_blocks;
  int batch, width, block_size, block_shift;  // shift: log2 of the block size, or -1
  long long num_tokens;  // rows of the outputs
  void *slots, *positions;  // OT [num_tokens]
  int *request_ids;         // [num_tokens]
  int *start;               // [B + 1]
  int *seq_lens;            // [B]
  int *taken;               // [B + 1]
  DeviceStatus *status;
};

// Rotary positions of q and k rows, k and v to their pages.
struct RopeArgs {
  const void *positions;  // PT [T]
  const void *slots;      // ST [T] or null
  const void *q, *k, *v;  // rows of H, KH, KH heads; null: none
  void *q_out, *k_out;    // null: not written
  void *k_cache, *v_cache;
  const void *table;  // CT [max_pos, rot]
  long long q_stride, k_stride, v_stride, q_out_stride, k_out_stride;  // elements per row
  long long k_block, k_slot, k_head, v_block, v_slot, v_head;          // cache strides
  long long num_slots, max_pos, num_tokens;
  int block_size, heads, kv_heads, dim, rot;
  bool neox, long_pos, long_slots;
  DeviceStatus *status;
};

// Paged keys: a prefix in the pages `prefix_blocks`, then each request's own
// keys in its row of `tables`.
struct PagedArgs {
  const void *q, *k, *v;  // q [B, Tq, H, D]; k, v [NB, BS, KH, D]
  void *out;              // [B, Tq, H, D] dense
  float *lse;             // [B, Tq, H] or null
  const int *prefix_blocks, *tables, *own_lens;
  const float *slopes;  // [H] or null
  long long q_batch, q_token, q_head;
  long long k_block, k_slot, k_head, v_block, v_slot, v_head;
  long long table_stride;
  long long prefix_len;
  int batch, q_len, heads, kv_heads, block_size, num_blocks, width;
  float scale, softcap;
  DeviceStatus *status;
};

// Dense keys at given positions.
struct PositionArgs {
  const void *q, *k, *v;  // q [Tq, H, D]; k, v [Tk, KH, D]
  void *out;              // [Tq, H, D] dense
  float *lse;             // [Tq, H] or null
  const void *q_pos, *k_pos;         // int32 or int64; k_pos null: 0, 1, 2, ...
  const int *q_doc, *k_doc;          // null: one document
  const int *q_prefix;               // null: none
  const float *slopes;
  long long q_token, q_head, k_token, k_head, v_token, v_head;
  int q_tokens, k_tokens, heads, kv_heads;
  bool long_q_pos, long_k_pos, causal;
  float scale, softcap;
};

// Which kernels an attention call takes, in slices of the keys (0: not taken).
struct PrefixPasses {
  int tensor_core, split_prefix, own;  // the prefix, or else in the own pass
};
struct PositionPasses {
  int tensor_core, split;  // one of them; tensor_core 1: whole, more: joined
};
PrefixPasses prefix_passes(const PagedArgs &a);
PositionPasses position_passes(const PositionArgs &a);

cudaError_t launch_slot_mapping(const SlotArgs &a, bool long_lens, bool long_slots,
                                cudaStream_t stream);
cudaError_t launch_rope_cache(const RopeArgs &a, RowType rows, RowType table, bool vec,
                              cudaStream_t stream);
// Bytes of device workspace (16-byte aligned) that a launch takes.
long long shared_prefix_attention_workspace(const PagedArgs &a, int dim);
cudaError_t launch_shared_prefix_attention(const PagedArgs &a, RowType type, int dim,
                                           void *workspace, cudaStream_t stream);
long long position_attention_workspace(const PositionArgs &a, int dim);
cudaError_t launch_position_attention(const PositionArgs &a, RowType type, int dim,
                                      void *workspace, cudaStream_t stream);

}  // namespace lmc
