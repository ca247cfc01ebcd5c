// Attention of few rows, or over few keys, split over the keys.
//
// A block owns 16 rows of one KV head (a request's query tokens and heads; a
// decode step's group of heads fits) and a slice of their keys.  Each of its
// four warps streams 16 keys at a time through its own ring of cp.async stages
// and keeps its own maximum, sum and output, so no barrier is met until the
// warps' results are joined at the end.  Products are 16x8x16 tensor
// instructions: the block reads every key and value once and multiplies it with
// 16 rows, 16 flop a byte, so it is bound by the reads and the small
// instruction loses nothing.  Any block size, page order and stride; dense keys
// for few rows or short calls, where the tensor-core kernel's 256-row blocks
// would wait most of the time.  Up to eight slices of a row are one cluster: its
// blocks join their parts through shared memory and write the result; more go
// through memory and a join kernel.
#pragma once
#include "attention_join.cuh"

namespace lmc {

constexpr int kSplitWarps = 4, kSplitKeys = 16, kSplitRows = 16, kSplitStages = 2;

// Which keys and rows a pass covers.  Paged: prefix keys [pre_begin, pre_end),
// then the own keys of the unit's request when `own`; a unit is a request, or all
// of them (own == false).  Dense: one unit of all rows, all keys.
struct SplitPass {
  int pre_begin, pre_end;
  bool own;
  int unit_tokens, row_tiles, slices, group;  // group: heads per KV head
  // first slice of this pass; null: write the result (the blocks of a row's slices
  // are then one cluster and join through shared memory)
  float *part_o, *part_lse;
};
constexpr int kMostClustered = 8;  // blocks of a cluster that every GPU takes

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::
                   : "memory");
}
// The same shared-memory place in block `rank` of the cluster.
__device__ __forceinline__ uint32_t in_block(uint32_t addr, int rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ float ld_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float2 ld_cluster2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr)
               : "memory");
  return v;
}

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
template <typename T>
__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                          uint32_t b1) {
  if constexpr (__is_same(T, __nv_bfloat16))
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <int D>
struct SplitSmem {
  static constexpr int kKeys = kSplitKeys * D * 2;        // 16 rows of K or V
  static constexpr int kStage = 2 * kKeys;
  static constexpr int kWarp = kSplitStages * kStage;
  static constexpr int kBytes = kSplitWarps * kWarp;
  // the join at the end: each warp's output and statistics, then the block's
  static_assert(kBytes >= (kSplitWarps + 1) * kSplitRows * (D + 2) * 4, "join fits in the rings");
};

// A row of the batch by the definition, on one warp: when a joined result holds
// an infinity or NaN (a draft token's value that earlier rows must not see).
template <typename T, int D>
__device__ __noinline__ void strict_paged_row(const PagedArgs &a, long long r) {
  const int h = static_cast<int>(r % a.heads), kv = h / (a.heads / a.kv_heads);
  const int t = static_cast<int>(r / a.heads), b = t / a.q_len, i = t - b * a.q_len;
  const int n = max(0, a.own_lens[b]);
  const long long pos = a.prefix_len + n - a.q_len + i;
  const long long room = static_cast<long long>(a.width) * a.block_size;
  const long long own = min(room, max(0ll, static_cast<long long>(n) - a.q_len + i + 1));
  const float slope = a.slopes ? a.slopes[h] : 0.f;
  WarpRow<T, D> row;
  row.start(static_cast<const T *>(a.q) + b * a.q_batch + i * a.q_token + h * a.q_head);
  const long long keys = a.prefix_len + own;
#pragma unroll 1
  for (long long j0 = 0; j0 < keys && !row.lost(); j0 += 32) {
    const long long j = min(j0 + (threadIdx.x & 31), keys - 1);
    const bool shared = j < a.prefix_len;
    const unsigned at = static_cast<unsigned>(shared ? j : j - a.prefix_len);
    const unsigned col = at / static_cast<unsigned>(a.block_size);
    const int off = static_cast<int>(at - col * a.block_size);
    int page = shared ? a.prefix_blocks[col] : a.tables[b * a.table_stride + col];
    const bool sees = j0 + (threadIdx.x & 31) < keys && page >= 0 && page < a.num_blocks;
    if (!sees) page = 0;
    row.add(sees, static_cast<const T *>(a.k) + page * a.k_block + off * a.k_slot + kv * a.k_head,
            static_cast<const T *>(a.v) + page * a.v_block + off * a.v_slot + kv * a.v_head,
            a.scale, a.softcap, slope * fabsf(static_cast<float>(pos - j)));
  }
  row.finish(static_cast<T *>(a.out) + r * D, a.lse ? a.lse + r : nullptr);
}

// kShaped: a cap or a distance bias.  Three blocks per SM: twelve warps with a
// stage each under way beat eight with two (64 requests on own keys of 64 to 1024,
// 120 MB: 38 us so).
template <typename T, int D, typename Args, bool kShaped>
__global__ void __launch_bounds__(kSplitWarps * 32, 3)
    split_attention_kernel(const __grid_constant__ Args a, const __grid_constant__ SplitPass s) {
  constexpr bool kDense = __is_same(Args, PositionArgs);
  using L = SplitSmem<D>;
  constexpr int kChunks = D / 8;  // 16-byte chunks of a row
  extern __shared__ __align__(128) uint8_t smem[];
  if (s.part_o != nullptr) let_next_start();  // a join or another pass follows
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int group = s.group, slice = blockIdx.y;
  // KV heads next to each other run together: their rows share DRAM pages
  const unsigned tile = blockIdx.x / static_cast<unsigned>(a.kv_heads);
  const int kv = blockIdx.x - tile * a.kv_heads;
  const int unit = s.row_tiles == 1 ? tile : tile / static_cast<unsigned>(s.row_tiles);
  const int row_tile = tile - unit * s.row_tiles;
  int n = 0, pre = 0, own_keys = 0, total;
  long long all_rows;
  if constexpr (kDense) {
    total = a.k_tokens;
    all_rows = static_cast<long long>(a.q_tokens) * a.heads;
  } else {
    // the pass's prefix part, then own keys within the request's table row
    n = s.own ? max(0, a.own_lens[unit]) : 0;
    pre = s.pre_end - s.pre_begin;
    const long long room = static_cast<long long>(a.width) * a.block_size;
    own_keys = static_cast<int>(min(static_cast<long long>(n), room));
    if (n > room && slice == 0 && row_tile == 0 && threadIdx.x == 0)
      report_status(a.status, kStatusBadIndex, unit, n, room);
    total = pre + own_keys;
    all_rows = static_cast<long long>(a.batch) * a.q_len * a.heads;
  }
  const int chunk = kSplitWarps * kSplitKeys;
  const int per = ((total + s.slices - 1) / s.slices + chunk - 1) / chunk * chunk;
  const int k0 = min(total, slice * per), k1 = min(total, k0 + per);

  // this lane's two rows of the tile, r0 and r1 (rows past the unit's are not
  // stored); the tile's result rows, -1 past the last
  __shared__ int result_row[kSplitRows];
  const int rows = min(kSplitRows, s.unit_tokens * group - row_tile * kSplitRows);
  const int r0 = lane >> 2, r1 = r0 + 8, c0 = (lane & 3) * 2;
  struct LaneRow {
    int token, head;
    bool valid;
  };
  auto lane_row = [&](int r) -> LaneRow {
    const int at = row_tile * kSplitRows + r, t = at / group;
    return {unit * s.unit_tokens + t, kv * group + at - t * group, r < rows};
  };
  const LaneRow row0 = lane_row(r0), row1 = lane_row(r1);
  if (threadIdx.x < 32 && (lane & 3) == 0) {
    result_row[r0] = row0.valid ? row0.token * a.heads + row0.head : -1;
    result_row[r1] = row1.valid ? row1.token * a.heads + row1.head : -1;
  }
  RawMask raw0 = {0, 0, 0}, raw1 = {0, 0, 0};
  if constexpr (kDense) {
    if (row0.valid) raw0 = load_mask(a, row0.token);
    if (row1.valid) raw1 = load_mask(a, row1.token);
  }
  float *part_o = s.part_o + static_cast<long long>(slice) * all_rows * D;
  float *part_lse = s.part_lse + static_cast<long long>(slice) * all_rows;
  const bool direct = s.part_o == nullptr;
  if (k0 >= k1 && !direct) {  // no keys: an empty part
    if (threadIdx.x < 32 && (lane & 3) == 0) {
      if (row0.valid) part_lse[result_row[r0]] = -INFINITY;
      if (row1.valid) part_lse[result_row[r1]] = -INFINITY;
    }
    wait_for_previous();
    return;
  }

  uint8_t *ring = smem + warp * L::kWarp;
  const uint32_t ring_addr = smem_u32(ring);
  const int steps = (k1 - k0 + chunk - 1) / chunk;

  // Where the 16 keys of step `it` of this warp lie, in elements from the first:
  // lane i (and i + 16) key i; -1 where there is none.  (Paged.)
  struct Place {
    long long k, v;
    bool bad;  // in a page outside the cache
  };
  auto place_of = [&](int it) -> Place {
    if constexpr (kDense) {
      return {0, 0, false};  // a row's place is its index
    } else {
      const int j = k0 + it * chunk + warp * kSplitKeys + (lane & 15);
      if (j >= k1) return {-1, -1, false};
      const bool shared = j < pre;
      const unsigned at = shared ? s.pre_begin + j : j - pre;
      const unsigned col = at / static_cast<unsigned>(a.block_size);
      const int off = static_cast<int>(at - col * a.block_size);
      const int page = shared ? a.prefix_blocks[col] : a.tables[unit * a.table_stride + col];
      if (page >= 0 && page < a.num_blocks)
        return {page * a.k_block + off * a.k_slot, page * a.v_block + off * a.v_slot, false};
      if (lane < 16) report_status(a.status, kStatusBadSlot, shared ? -1 : unit, col, page);
      return {-1, -1, true};
    }
  };
  const T *k_first = static_cast<const T *>(a.k) + kv * a.k_head + lane % kChunks * 8;
  const T *v_first = static_cast<const T *>(a.v) + kv * a.v_head + lane % kChunks * 8;
  bool alike;  // K and V rows lie at the same offsets
  if constexpr (kDense)
    alike = a.k_token == a.v_token;
  else
    alike = a.k_block == a.v_block && a.k_slot == a.v_slot;
  auto load = [&](int it, const Place &p) {
    const uint32_t dst = ring_addr + (it % kSplitStages) * L::kStage;
    const int c = lane % kChunks;
    constexpr int kRowsAtOnce = 32 / kChunks;
    const int j0 = k0 + it * chunk + warp * kSplitKeys;
#pragma unroll
    for (int i = 0; i < kSplitKeys / kRowsAtOnce; ++i) {
      const int r = i * kRowsAtOnce + lane / kChunks;
      long long ko, vo;
      bool valid;  // else zeros: nothing is read
      if constexpr (kDense) {
        valid = j0 + r < k1;
        ko = (j0 + r) * a.k_token, vo = alike ? ko : (j0 + r) * a.v_token;
      } else {
        ko = __shfl_sync(0xffffffffu, p.k, r);
        vo = alike ? ko : __shfl_sync(0xffffffffu, p.v, r);
        valid = ko >= 0;
      }
      const uint32_t at = r * (D * 2) + ((c & ~7) << 4) + (((c & 7) ^ (r & 7)) << 4);
      cp_async16(dst + at, k_first + (valid ? ko : 0), valid);
      cp_async16(dst + L::kKeys + at, v_first + (valid ? vo : 0), valid);
    }
  };

  // keys of each stage in flight that lie outside the cache
  uint32_t bad_ring[kSplitStages];
#pragma unroll
  for (int i = 0; i < kSplitStages; ++i) bad_ring[i] = 0;
  Place next = {-1, -1, false};
#pragma unroll
  for (int i = 0; i < kSplitStages - 1; ++i) {
    if (i < steps) {
      next = place_of(i);
      bad_ring[i] = __ballot_sync(0xffffffffu, next.bad) & 0xffff;
      load(i, next);
    }
    cp_async_commit();
  }
  next = {-1, -1, false};
  if (kSplitStages - 1 < steps) next = place_of(kSplitStages - 1);

  // Q as the A operand: row lane/4 (and + 8), columns 2 (lane % 4) of each 8.
  uint32_t q[D / 16][4];
  auto q_row = [&](const LaneRow &r) -> const T * {
    if (!r.valid) return nullptr;
    const T *p = static_cast<const T *>(a.q) + r.head * a.q_head;
    if constexpr (kDense) return p + r.token * a.q_token;
    else return p + r.token / a.q_len * a.q_batch + r.token % a.q_len * a.q_token;
  };
  {
    const T *p0 = q_row(row0), *p1 = q_row(row1);
#pragma unroll
    for (int k = 0; k < D / 16; ++k) {
      const int c = k * 16 + c0;
      q[k][0] = p0 ? *reinterpret_cast<const uint32_t *>(p0 + c) : 0;
      q[k][1] = p1 ? *reinterpret_cast<const uint32_t *>(p1 + c) : 0;
      q[k][2] = p0 ? *reinterpret_cast<const uint32_t *>(p0 + c + 8) : 0;
      q[k][3] = p1 ? *reinterpret_cast<const uint32_t *>(p1 + c + 8) : 0;
    }
  }
  // Paged: row i of a request sees its own keys up to n - q_len + i, as an index
  // into this pass's keys j < last.  Dense: positions below the row's limit in its
  // document.
  RowMask mask0 = {0, 0, 0}, mask1 = {0, 0, 0};
  int last0 = total, last1 = total;
  float slope0 = 0.f, slope1 = 0.f;
  long long at0 = 0, at1 = 0;  // paged rows' positions
  if (a.slopes) {
    slope0 = row0.valid ? a.slopes[row0.head] * kLog2e : 0.f;
    slope1 = row1.valid ? a.slopes[row1.head] * kLog2e : 0.f;
  }
  if constexpr (kDense) {
    mask0 = row_mask(a, raw0);
    mask1 = row_mask(a, raw1);
  } else {
    auto place = [&](const LaneRow &r, int &last, long long &at) {
      if (!r.valid) return;
      const int b = s.own ? unit : r.token / a.q_len, i = r.token - b * a.q_len;
      if (s.own) last = pre + max(0, min(own_keys, n - a.q_len + i + 1));
      if (a.slopes) at = a.prefix_len + max(0, a.own_lens[b]) - a.q_len + i;
    };
    place(row0, last0, at0);
    place(row1, last1, at1);
  }
  // keys below this index, position and document are seen by all of the tile's rows
  int all_last = 0, all_limit = 0;
  if constexpr (kDense)
    all_limit = __reduce_min_sync(0xffffffffu, min(row0.valid ? mask0.limit : 2147483647,
                                                   row1.valid ? mask1.limit : 2147483647));
  else
    all_last = __reduce_min_sync(0xffffffffu, min(min(last0, last1), k1));
  // -slope times the distance between the row and pass key j
  auto bias = [&](bool second, int j, int kp) {
    if constexpr (kDense) {
      const long long at = second ? mask1.pos : mask0.pos;
      return -(second ? slope1 : slope0) * fabsf(static_cast<float>(at - kp));
    } else {
      const long long at = j < pre ? s.pre_begin + j : a.prefix_len + (j - pre);
      return -(second ? slope1 : slope0) *
             fabsf(static_cast<float>((second ? at1 : at0) - at));
    }
  };
  // dense: position and document of key lane % 16 of a step
  int kp_next = 0, kd_next = 0;
  auto key_marks = [&](int it) {
    if constexpr (kDense) {
      const int j = min(k0 + it * chunk + warp * kSplitKeys + (lane & 15), a.k_tokens - 1);
      kp_next = a.k_pos ? clamp_pos(position_at(a.k_pos, a.long_k_pos, j)) : j;
      kd_next = a.k_doc ? a.k_doc[j] : 0;
    }
  };
  if (steps > 0) key_marks(0);
  const float scale = a.scale * kLog2e;
  const float cap_u = a.softcap > 0.f ? a.scale / a.softcap : 0.f;
  const float cap_in = 2.f * kLog2e * cap_u;
  const float cap_out = a.softcap * kLog2e;

  float o[D / 8][4];
#pragma unroll
  for (int d = 0; d < D / 8; ++d) o[d][0] = o[d][1] = o[d][2] = o[d][3] = 0.f;
  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;

  for (int it = 0; it < steps; ++it) {
    // one more step's loads, and the pages of the step after it
    {
      const int nx = it + kSplitStages - 1;
      __syncwarp();  // every lane is done with the stage that is filled next
      if (nx < steps) {
        const uint32_t b = __ballot_sync(0xffffffffu, next.bad) & 0xffff;
#pragma unroll
        for (int i = 0; i < kSplitStages; ++i)
          if (nx % kSplitStages == i) bad_ring[i] = b;
        load(nx, next);
      }
      cp_async_commit();
      if (nx + 1 < steps) next = place_of(nx + 1);
    }
    const int kp_all = kp_next, kd_all = kd_next;
    if (it + 1 < steps) key_marks(it + 1);
    cp_async_wait<kSplitStages - 1>();
    __syncwarp();
    const uint32_t kb = ring_addr + (it % kSplitStages) * L::kStage, vb = kb + L::kKeys;
    float sc[2][4], odd[2][4];  // two chains of products each
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) sc[t][e] = odd[t][e] = 0.f;
#pragma unroll
    for (int k = 0; k < D / 16; ++k) {
      const int r = (lane & 7) + ((lane >> 4) << 3), c = k * 2 + ((lane >> 3) & 1);
      uint32_t b[4];
      ldmatrix4(b, kb + r * (D * 2) + ((c & ~7) << 4) + (((c & 7) ^ (r & 7)) << 4));
      mma_16816<T>(k & 1 ? odd[0] : sc[0], q[k], b[0], b[1]);
      mma_16816<T>(k & 1 ? odd[1] : sc[1], q[k], b[2], b[3]);
    }
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) sc[t][e] += odd[t][e];
    const int j0 = k0 + it * chunk + warp * kSplitKeys;
    uint32_t bad_keys = 0;
#pragma unroll
    for (int i = 0; i < kSplitStages; ++i)
      if (it % kSplitStages == i) bad_keys = bad_ring[i];
    if constexpr (kShaped) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int col = t * 8 + c0 + (e & 1);
          float x = sc[t][e];
          if (cap_out > 0.f) {
            // tanh(u) = 1 - 2 / (1 + e^2u) is off by some 2^-22 of the cap: below
            // u = 1/8 the series (next term 1.3e-9 of u)
            const float u = x * cap_u, w = u * u;
            const float small = fmaf(fmaf(fmaf(-17.f / 315.f, w, 2.f / 15.f), w, -1.f / 3.f), w, 1.f);
            x = fabsf(u) < 0.125f ? x * scale * small
                                  : fmaf(rcp(1.f + ex2(x * cap_in)), -2.f * cap_out, cap_out);
          } else {
            x *= scale;
          }
          const int kp = kDense ? __shfl_sync(0xffffffffu, kp_all, col) : 0;
          if (a.slopes) x += bias(e >= 2, j0 + col, kp);
          sc[t][e] = x;
        }
      }
    } else {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[t][e] *= scale;
    }
    bool open;  // no key of this step is masked for any row
    if constexpr (kDense)
      open = j0 + kSplitKeys <= k1 && a.k_doc == nullptr &&
             __reduce_max_sync(0xffffffffu, kp_all) < all_limit;
    else
      open = j0 + kSplitKeys <= all_last && bad_keys == 0;
    uint32_t sees = open ? 3 : 0;  // which of its rows see one of this lane's keys
    if (!open) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int col = t * 8 + c0 + e, j = j0 + col;
          bool out0 = j >= k1, out1 = out0;
          if constexpr (kDense) {
            const int kp = __shfl_sync(0xffffffffu, kp_all, col);
            const int kd = __shfl_sync(0xffffffffu, kd_all, col);
            out0 = out0 || kp >= mask0.limit || (a.k_doc && kd != mask0.doc);
            out1 = out1 || kp >= mask1.limit || (a.k_doc && kd != mask1.doc);
          } else {
            const bool bad_key = (bad_keys >> col) & 1;
            out0 = out0 || j >= last0 || bad_key;
            out1 = out1 || j >= last1 || bad_key;
          }
          if (out0) sc[t][e] = -INFINITY;
          if (out1) sc[t][2 + e] = -INFINITY;
          sees |= (out0 ? 0 : 1) | (out1 ? 0 : 2);  // (as two flags: 4% of a short call)
        }
      }
    }
    float top0 = fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[1][0], sc[1][1]));
    float top1 = fmaxf(fmaxf(sc[0][2], sc[0][3]), fmaxf(sc[1][2], sc[1][3]));
#pragma unroll
    for (int x = 1; x < 4; x <<= 1) {
      top0 = fmaxf(top0, __shfl_xor_sync(0xffffffffu, top0, x));
      top1 = fmaxf(top1, __shfl_xor_sync(0xffffffffu, top1, x));
    }
    const bool grow0 = top0 > m0 + kLazy, grow1 = top1 > m1 + kLazy;
    if (__any_sync(0xffffffffu, grow0 || grow1)) {
      const float to0 = grow0 ? top0 : m0, to1 = grow1 ? top1 : m1;
      const float f0 = grow0 ? ex2(m0 - to0) : 1.f, f1 = grow1 ? ex2(m1 - to1) : 1.f;
      m0 = to0, m1 = to1;
      l0 *= f0, l1 *= f1;
#pragma unroll
      for (int d = 0; d < D / 8; ++d) o[d][0] *= f0, o[d][1] *= f0, o[d][2] *= f1, o[d][3] *= f1;
    }
    // no finite score yet: zero weights, or NaN ones for keys that are seen and have
    // scores of -inf (they lead the row to the definition)
    const float off0 = (m0 == -INFINITY && !(sees & 1) ? 0.f : m0) - kRaised<T>;
    const float off1 = (m1 == -INFINITY && !(sees & 2) ? 0.f : m1) - kRaised<T>;
    uint32_t p[4];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const float w0 = ex2(sc[t][0] - off0), w1 = ex2(sc[t][1] - off0);
      const float w2 = ex2(sc[t][2] - off1), w3 = ex2(sc[t][3] - off1);
      l0 += w0 + w1, l1 += w2 + w3;
      p[2 * t] = pair_from_float<T>(w0, w1);
      p[2 * t + 1] = pair_from_float<T>(w2, w3);
    }
#pragma unroll
    for (int d = 0; d < D / 16; ++d) {
      const int r = (lane & 7) + (((lane >> 3) & 1) << 3), c = d * 2 + (lane >> 4);
      uint32_t b[4];
      ldmatrix4_trans(b, vb + r * (D * 2) + ((c & ~7) << 4) + (((c & 7) ^ (r & 7)) << 4));
      mma_16816<T>(o[2 * d], p, b[0], b[1]);
      mma_16816<T>(o[2 * d + 1], p, b[2], b[3]);
    }
  }
  // --- the four warps' results in one
#pragma unroll
  for (int x = 1; x < 4; x <<= 1) {
    l0 += __shfl_xor_sync(0xffffffffu, l0, x);
    l1 += __shfl_xor_sync(0xffffffffu, l1, x);
  }
  cp_async_wait<0>();
  __syncthreads();
  float *wo = reinterpret_cast<float *>(smem);                 // [warp][16][D]
  float *wm = wo + kSplitWarps * kSplitRows * D;               // [warp][16]
  float *wl = wm + kSplitWarps * kSplitRows;
  if ((lane & 3) == 0) {
    wm[warp * kSplitRows + r0] = m0, wm[warp * kSplitRows + r1] = m1;
    wl[warp * kSplitRows + r0] = l0, wl[warp * kSplitRows + r1] = l1;
  }
#pragma unroll
  for (int d = 0; d < D / 8; ++d) {
    float *w0 = wo + (warp * kSplitRows + r0) * D + d * 8 + c0;
    *reinterpret_cast<float2 *>(w0) = make_float2(o[d][0], o[d][1]);
    *reinterpret_cast<float2 *>(w0 + 8 * D) = make_float2(o[d][2], o[d][3]);
  }
  __syncthreads();
  constexpr int kEach = D / 32;  // elements of a lane
  uint32_t again = 0;
  // a row's result from its sum, the sum of its weights and their maximum
  auto write = [&](int i, int row, float (&acc)[kEach], float m, float l) {
    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : NAN);
    bool finite = true;
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      acc[e] *= inv;
      finite = finite && fabsf(acc[e]) <= 3.4028235e38f;
    }
    const long long at = static_cast<long long>(row) * D + lane * kEach;
#pragma unroll
    for (int e = 0; e < kEach / 2; ++e) {
      if (direct)
        reinterpret_cast<uint32_t *>(static_cast<T *>(a.out) + at)[e] =
            pair_from_float<T>(acc[2 * e], acc[2 * e + 1]);
      else
        reinterpret_cast<float2 *>(part_o + at)[e] = make_float2(acc[2 * e], acc[2 * e + 1]);
    }
    if (lane == 0) {
      const float log2_sum = log2_of_sum(true, m - kRaised<T>, l);
      if (!direct) part_lse[row] = log2_sum;
      else if (a.lse) a.lse[row] = log2_sum * kLn2;
    }
    if (direct && !__all_sync(0xffffffffu, finite)) again |= 1u << i;
  };
  const bool clustered = direct && s.slices > 1;
  float *bo = wl + kSplitWarps * kSplitRows;  // the block's [16][D], maxima and sums
  float *bm = bo + kSplitRows * D, *bl = bm + kSplitRows;
  auto finish = [&](int i) {
    const int r = warp + i * kSplitWarps;
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int w = 0; w < kSplitWarps; ++w) m = fmaxf(m, wm[w * kSplitRows + r]);
    const float base = m == -INFINITY ? 0.f : m;
    float f[kSplitWarps];
#pragma unroll
    for (int w = 0; w < kSplitWarps; ++w) {
      f[w] = ex2(wm[w * kSplitRows + r] - base);
      l = fmaf(f[w], wl[w * kSplitRows + r], l);
    }
    float acc[kEach];
#pragma unroll
    for (int e = 0; e < kEach; ++e) acc[e] = 0.f;
#pragma unroll
    for (int w = 0; w < kSplitWarps; ++w) {
      const float2 *v = reinterpret_cast<const float2 *>(wo + (w * kSplitRows + r) * D + lane * kEach);
#pragma unroll
      for (int e = 0; e < kEach / 2; ++e) {
        acc[2 * e] = fmaf(f[w], v[e].x, acc[2 * e]);
        acc[2 * e + 1] = fmaf(f[w], v[e].y, acc[2 * e + 1]);
      }
    }
    if (clustered) {
#pragma unroll
      for (int e = 0; e < kEach / 2; ++e)
        reinterpret_cast<float2 *>(bo + r * D + lane * kEach)[e] =
            make_float2(acc[2 * e], acc[2 * e + 1]);
      if (lane == 0) bm[r] = m, bl[r] = l;
    } else if (result_row[r] >= 0) {
      write(i, result_row[r], acc, m, l);
    }
  };
  finish(0);
  if (rows > kSplitWarps) {
    // side by side: one row after the other they cost more than two steps
#pragma unroll
    for (int i = 1; i < kSplitRows / kSplitWarps; ++i) finish(i);
  }
  if (clustered) {
    // the rows are dealt to the cluster's blocks, which read the others' parts
    cluster_sync();
    for (int i = 0, r = slice * kSplitWarps + warp; r < rows; ++i, r += s.slices * kSplitWarps) {
      const uint32_t m_at = smem_u32(bm + r), l_at = smem_u32(bl + r);
      const uint32_t o_at = smem_u32(bo + r * D + lane * kEach);
      float ms[kMostClustered], m = -INFINITY, l = 0.f, acc[kEach];
#pragma unroll
      for (int b = 0; b < kMostClustered; ++b) {
        ms[b] = b < s.slices ? ld_cluster(in_block(m_at, b)) : -INFINITY;
        m = fmaxf(m, ms[b]);
      }
      const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int e = 0; e < kEach; ++e) acc[e] = 0.f;
#pragma unroll
      for (int b = 0; b < kMostClustered; ++b) {
        if (b >= s.slices) continue;
        const float f = ex2(ms[b] - base);
        l = fmaf(f, ld_cluster(in_block(l_at, b)), l);
#pragma unroll
        for (int e = 0; e < kEach / 2; ++e) {
          const float2 v = ld_cluster2(in_block(o_at, b) + e * 8);
          acc[2 * e] = fmaf(f, v.x, acc[2 * e]);
          acc[2 * e + 1] = fmaf(f, v.y, acc[2 * e + 1]);
        }
      }
      write(i, result_row[r], acc, m, l);
    }
    cluster_sync();  // no block leaves while another reads its memory
  }
  if (again) {
    __syncwarp();  // the rows written above are written again
    for (int i = 0; i < kSplitRows / kSplitWarps; ++i) {
      if (!((again >> i) & 1)) continue;
      const int row = result_row[clustered ? (i * s.slices + slice) * kSplitWarps + warp
                                           : warp + i * kSplitWarps];
      if constexpr (kDense)
        strict_position_row<T, D>(a, row / a.heads, row % a.heads);
      else
        strict_paged_row<T, D>(a, row);
    }
  }
  wait_for_previous();
}

// Towards one wave of three blocks per SM, with 128 keys or more each; eight parts
// rather than up to sixteen, because a cluster joins them in the same launch.
// Measured (us, 8 KV heads of 128): 16 requests on 500 tokens 15.8 in one part, 11.0
// in parts of 128; one row on 1024 keys 19.4 / 6.9.  Between 256 and 384 keys two
// parts pay while their blocks have an SM each (one / two parts, 260 keys: 72 blocks
// 9.1 / 8.6, 80 blocks 9.2 / 10.2, 200 blocks 11.6 / 12.5; D 64 7.0 / 7.0, 7.0 / 7.7,
// 8.3 / 9.1; capped 11.1 / 10.1, 11.0 / 11.5, 13.6 / 14.6; 383 keys alike).  A deeper
// ring (six stages) changed none of these: a step's own chain of instructions takes
// its 0.8 us.
inline int split_slices(long long blocks, long long keys) {
  if (keys < 256 || (keys < 384 && blocks > 74)) return 1;
  long long want = std::min(444 / std::max(1ll, blocks), keys / 128);
  if (want > kMostClustered && want <= 2 * kMostClustered) want = kMostClustered;
  return static_cast<int>(std::max(1ll, std::min(want, 64ll)));
}

template <typename T, int D, typename Args>
cudaError_t launch_split(const Args &a, const SplitPass &s, long long units, bool first,
                         cudaStream_t stream) {
  constexpr int kBytes = SplitSmem<D>::kBytes;
  auto kernel = a.softcap > 0.f || a.slopes != nullptr
                    ? split_attention_kernel<T, D, Args, true>
                    : split_attention_kernel<T, D, Args, false>;
  cudaError_t e = allow_smem(kernel, kBytes);
  if (e != cudaSuccess) return e;
  const dim3 grid(static_cast<unsigned>(units * s.row_tiles * a.kv_heads), s.slices);
  return launch_ordered(kernel, grid, kSplitWarps * 32, kBytes, first, stream,
                        s.part_o == nullptr ? s.slices : 1, a, s);
}

template <typename T, int D>
__global__ void __launch_bounds__(128)
    join_paged_kernel(const __grid_constant__ PagedArgs a, const float *part_o,
                      const float *part_lse, int slices) {
  const long long rows = static_cast<long long>(a.batch) * a.q_len * a.heads;
  const long long row = static_cast<long long>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  wait_for_previous();
  if (row >= rows) return;
  JoinedRow<T, D> r;
  r.join(part_o, part_lse, slices, rows, row);
  if (r.finite())
    r.store(static_cast<T *>(a.out), a.lse, row);
  else
    strict_paged_row<T, D>(a, row);
}

}  // namespace lmc
