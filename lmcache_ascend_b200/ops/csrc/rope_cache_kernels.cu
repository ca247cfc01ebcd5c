// Rotary positions of fresh queries and keys, with K and V written to their
// pages in the same pass.
//
// A head's first `rot` elements are rotated in pairs by the angle of the row's
// position, y1 = x1 cos - x2 sin and y2 = x2 cos + x1 sin, in fp32 with one
// rounding to the row's type; the rest of the head passes through.  Pairs are
// (i, i + rot/2) in the half layout ("neox") and (2i, 2i + 1) interleaved.  The
// table row of a position holds rot/2 cosines and rot/2 sines (a scaled table,
// with its gain, is used as it is).
//
// Bound by HBM: each row is read once and written once, so K and V go straight
// to their slots instead of through a second pass.  A thread moves units of two
// 16-byte vectors that hold both halves of its pairs (in the half layout the
// vectors at i and i + rot/2, otherwise two adjacent ones); a head of D elements
// has D / (2 * VE) units whatever the layout.  A thread keeps its place in the
// head and walks over the heads of q, k and v of one row after the other, so that
// a unit costs no division and a row's cosines and sines are loaded once for
// several heads; blocks get equal work for one row or many.  The loads in flight
// come from many threads with one unit each (five blocks of 256 per SM), not from
// several units a thread: 16385 rows of 64/8 heads of 128 (680 MB) take 117 us
// (5.8 TB/s) so, 150 us with two units a thread in four blocks, 126 us in six
// blocks (spills).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "common.cuh"
#include "serving_ops.h"

namespace lmc {
namespace {

constexpr int kRopeThreads = 256;
constexpr int kHeadsPerThread = 12, kBlockHeads = 2048, kResident = 148 * 5;

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float as_float(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T round_to(float v);
template <>
__device__ __forceinline__ float round_to<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 round_to<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half round_to<__half>(float v) { return __float2half_rn(v); }

__device__ __forceinline__ long long int_at(const void *p, bool is_long, long long i) {
  return is_long ? static_cast<const long long *>(p)[i]
                 : static_cast<long long>(static_cast<const int *>(p)[i]);
}

// Which head a row's flat head index names, and where its result goes.
template <typename T>
struct HeadRef {
  const T *src;
  T *dst, *dst2;  // either may be null
  bool rotate;
};

template <typename T>
__device__ __forceinline__ HeadRef<T> head_ref(const RopeArgs &a, long long t, int h) {
  HeadRef<T> r = {nullptr, nullptr, nullptr, true};
  if (h < a.heads) {
    r.src = static_cast<const T *>(a.q) + t * a.q_stride + static_cast<long long>(h) * a.dim;
    r.dst = static_cast<T *>(a.q_out) + t * a.q_out_stride + static_cast<long long>(h) * a.dim;
    return r;
  }
  h -= a.heads;
  const bool is_k = h < a.kv_heads;
  if (!is_k) h -= a.kv_heads;
  r.rotate = is_k;
  r.src = is_k ? static_cast<const T *>(a.k) + t * a.k_stride : static_cast<const T *>(a.v) +
                                                                    t * a.v_stride;
  r.src += static_cast<long long>(h) * a.dim;
  if (is_k && a.k_out)
    r.dst = static_cast<T *>(a.k_out) + t * a.k_out_stride + static_cast<long long>(h) * a.dim;
  if (a.slots) {
    const long long slot = int_at(a.slots, a.long_slots, t);
    if (slot >= 0 && slot < a.num_slots) {
      const unsigned page = static_cast<unsigned>(slot / a.block_size);
      const int off = static_cast<int>(slot - static_cast<long long>(page) * a.block_size);
      r.dst2 = is_k ? static_cast<T *>(a.k_cache) + page * a.k_block + off * a.k_slot +
                          h * a.k_head
                    : static_cast<T *>(a.v_cache) + page * a.v_block + off * a.v_slot +
                          h * a.v_head;
    } else if (slot >= a.num_slots) {
      report_status(a.status, kStatusBadSlot, 0, t, slot);
    }
  }
  return r;
}

template <typename CT, int N>
__device__ __forceinline__ void load_table(const CT *p, float *f) {
  // (wider vectors than N are never launched: the launcher checks)
  constexpr int V = 16 / sizeof(CT) < N ? 16 / sizeof(CT) : N;
#pragma unroll
  for (int i = 0; i < N; i += V) {
    const uint4 w = __ldg(reinterpret_cast<const uint4 *>(p + i));  // the table is not written
    const CT *e = reinterpret_cast<const CT *>(&w);
#pragma unroll
    for (int j = 0; j < V; ++j) f[i + j] = as_float(e[j]);
  }
}

// 16-byte units.  Needs dim % (2 VE) == 0 and rot % (2 VE) == 0, aligned rows and
// at most kRopeThreads units per head.  `heads` counts those of q, k and v; a
// block takes `per_block` of them in a row, up to kHeadsPerThread a thread.  Its
// rows are looked up first (position, page), so that its data and table loads wait
// for nothing but their own memory.
template <typename T, typename CT>
__global__ void __launch_bounds__(kRopeThreads, 5)
    rope_cache_vec_kernel(RopeArgs a, int heads, int per_block) {
  constexpr int VE = 16 / sizeof(T);
  struct Row {
    long long pos, k_at, v_at;  // position, offsets of the slot's first head; -1: none
  };
  extern __shared__ __align__(16) unsigned char rope_smem[];
  Row *rows = reinterpret_cast<Row *>(rope_smem);
  const int per_head = a.dim / (2 * VE);
  const int lanes = kRopeThreads / per_head;
  const long long total = a.num_tokens * heads;
  const long long first = static_cast<long long>(blockIdx.x) * per_block;
  const long long t_first = first / heads;
  const int rem = static_cast<int>(first - t_first * heads);
  const int count = static_cast<int>(min(total - first, static_cast<long long>(per_block)));
  const int n_rows = (rem + count - 1) / heads + 1;
  for (int i = threadIdx.x; i < n_rows; i += kRopeThreads) {
    const long long t = t_first + i;
    Row r = {int_at(a.positions, a.long_pos, t), -1, -1};
    if (r.pos < 0 || r.pos >= a.max_pos) {
      // no angle: nothing reaches the pages, the row's outputs are zero
      report_status(a.status, kStatusBadIndex, 0, t, r.pos);
      r.pos = -1;
    } else if (a.slots) {
      const long long slot = int_at(a.slots, a.long_slots, t);
      if (slot >= 0 && slot < a.num_slots) {
        const long long page = slot / a.block_size, off = slot - page * a.block_size;
        r.k_at = page * a.k_block + off * a.k_slot;
        r.v_at = page * a.v_block + off * a.v_slot;
      } else if (slot >= a.num_slots) {
        report_status(a.status, kStatusBadSlot, 0, t, slot);
      }
    }
    rows[i] = r;
  }
  __syncthreads();
  const int lane = static_cast<int>(threadIdx.x) / per_head;
  const int j = static_cast<int>(threadIdx.x) - lane * per_head;
  if (lane >= lanes) return;
  const bool rotated = j < a.rot / (2 * VE);
  int at1 = j * 2 * VE, at2 = at1 + VE;
  if (a.neox && rotated) at1 = j * VE, at2 = at1 + a.rot / 2;
  int dt = 0, h = rem + lane;  // row and head
  int angle_of = -1;           // row whose cosines and sines are in c and s
  float c[VE], s[VE];
#pragma unroll 1
  for (int done = lane; done < count; done += lanes, h += lanes) {
    while (h >= heads) h -= heads, ++dt;
    const long long t = t_first + dt;
    const Row &r = rows[dt];
    const T *src;
    T *dst = nullptr, *dst2 = nullptr;
    int of = h;
    bool turn = rotated;
    if (of < a.heads) {
      src = static_cast<const T *>(a.q) + t * a.q_stride + of * a.dim;
      dst = static_cast<T *>(a.q_out) + t * a.q_out_stride + of * a.dim;
    } else if ((of -= a.heads) < a.kv_heads) {
      src = static_cast<const T *>(a.k) + t * a.k_stride + of * a.dim;
      if (a.k_out) dst = static_cast<T *>(a.k_out) + t * a.k_out_stride + of * a.dim;
      if (r.k_at >= 0) dst2 = static_cast<T *>(a.k_cache) + r.k_at + of * a.k_head;
    } else {
      of -= a.kv_heads;
      turn = false;
      src = static_cast<const T *>(a.v) + t * a.v_stride + of * a.dim;
      if (r.v_at >= 0) dst2 = static_cast<T *>(a.v_cache) + r.v_at + of * a.v_head;
    }
    uint4 x = *reinterpret_cast<const uint4 *>(src + at1);
    uint4 y = *reinterpret_cast<const uint4 *>(src + at2);
    if (r.pos < 0) {
      x = y = make_uint4(0, 0, 0, 0);
    } else if (turn) {
      if (dt != angle_of) {
        const CT *table = static_cast<const CT *>(a.table) + r.pos * a.rot + j * VE;
        load_table<CT, VE>(table, c);
        load_table<CT, VE>(table + a.rot / 2, s);
        angle_of = dt;
      }
      T *p = reinterpret_cast<T *>(&x), *q = reinterpret_cast<T *>(&y);
      if (a.neox) {
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          const float f = as_float(p[e]), g = as_float(q[e]);
          p[e] = round_to<T>(f * c[e] - g * s[e]);
          q[e] = round_to<T>(g * c[e] + f * s[e]);
        }
      } else {
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          T *w = e < VE / 2 ? p + 2 * e : q + 2 * e - VE;
          const float f = as_float(w[0]), g = as_float(w[1]);
          w[0] = round_to<T>(f * c[e] - g * s[e]);
          w[1] = round_to<T>(g * c[e] + f * s[e]);
        }
      }
    }
    if (dst) {
      *reinterpret_cast<uint4 *>(dst + at1) = x;
      *reinterpret_cast<uint4 *>(dst + at2) = y;
    }
    if (dst2) {
      *reinterpret_cast<uint4 *>(dst2 + at1) = x;
      *reinterpret_cast<uint4 *>(dst2 + at2) = y;
    }
  }
}

// One pair of elements per thread: rows, pages or a rotated part that 16-byte
// units do not fit.  The same arithmetic, so the same bits.
template <typename T, typename CT>
__global__ void __launch_bounds__(kRopeThreads) rope_cache_pair_kernel(RopeArgs a) {
  const int per_head = (a.dim + 1) / 2;  // an odd head ends in a single element
  const int rot_pairs = a.rot / 2;
  const int per_row = per_head * (a.heads + (a.k ? a.kv_heads : 0) + (a.v ? a.kv_heads : 0));
  const long long total = a.num_tokens * per_row;
  for (long long u = static_cast<long long>(blockIdx.x) * kRopeThreads + threadIdx.x; u < total;
       u += static_cast<long long>(gridDim.x) * kRopeThreads) {
    const long long t = u / per_row;
    const int v = static_cast<int>(u - t * per_row);
    const int h = v / per_head, j = v - h * per_head;
    HeadRef<T> ref = head_ref<T>(a, t, h);
    const long long pos = int_at(a.positions, a.long_pos, t);
    int at1, at2;
    if (a.neox && j < rot_pairs)
      at1 = j, at2 = j + rot_pairs;
    else
      at1 = 2 * j, at2 = 2 * j + 1;
    const bool two = at2 < a.dim;
    T x = ref.src[at1], y = two ? ref.src[at2] : x;
    if (pos < 0 || pos >= a.max_pos) {
      report_status(a.status, kStatusBadIndex, 0, t, pos);
      x = y = round_to<T>(0.f);
      ref.dst2 = nullptr;
    } else if (ref.rotate && j < rot_pairs) {
      const CT *row = static_cast<const CT *>(a.table) + pos * a.rot + j;
      const float c = as_float(row[0]), s = as_float(row[rot_pairs]);
      const float f = as_float(x), g = as_float(y);
      x = round_to<T>(f * c - g * s);
      y = round_to<T>(g * c + f * s);
    }
    if (ref.dst) {
      ref.dst[at1] = x;
      if (two) ref.dst[at2] = y;
    }
    if (ref.dst2) {
      ref.dst2[at1] = x;
      if (two) ref.dst2[at2] = y;
    }
  }
}

template <typename T, typename CT>
cudaError_t launch(const RopeArgs &a, bool vec, cudaStream_t stream) {
  const long long heads = a.heads + (a.k ? a.kv_heads : 0) + (a.v ? a.kv_heads : 0);
  if (vec) {
    const long long lanes = kRopeThreads / (a.dim / (2 * (16 / static_cast<int>(sizeof(T)))));
    // heads a thread: whole waves of the blocks that fit, none much longer than
    // kHeadsPerThread (5001 rows of 48 heads: one wave of 11 each 26.8 us, 8 each 31)
    const long long all = a.num_tokens * heads;
    const long long most = std::min(1ll * kHeadsPerThread, kBlockHeads / lanes);
    const long long waves = (all + lanes * kResident * most - 1) / (lanes * kResident * most);
    const long long deep = (all + lanes * kResident * waves - 1) / (lanes * kResident * waves);
    const long long per_block = lanes * deep;
    const long long blocks = (all + per_block - 1) / per_block;
    if (blocks > 0x7fffffff) return cudaErrorInvalidConfiguration;
    const int rows = static_cast<int>((per_block + heads - 2) / heads + 1);  // at most, of a block
    rope_cache_vec_kernel<T, CT>
        <<<static_cast<unsigned>(blocks), kRopeThreads, rows * 24, stream>>>(
            a, static_cast<int>(heads), static_cast<int>(per_block));
  } else {
    const long long units = a.num_tokens * heads * ((a.dim + 1) / 2);
    const long long blocks = std::min((units + kRopeThreads - 1) / kRopeThreads, 148ll * 32);
    rope_cache_pair_kernel<T, CT><<<static_cast<unsigned>(blocks), kRopeThreads, 0, stream>>>(a);
  }
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch_table(const RopeArgs &a, RowType table, bool vec, cudaStream_t stream) {
  if (table == RowType::kFloat) return launch<T, float>(a, vec, stream);
  if (table == RowType::kBFloat16) return launch<T, __nv_bfloat16>(a, vec, stream);
  return launch<T, __half>(a, vec, stream);
}

}  // namespace

cudaError_t launch_rope_cache(const RopeArgs &a, RowType rows, RowType table, bool vec,
                              cudaStream_t stream) {
  if (rows == RowType::kFloat) return launch_table<float>(a, table, vec, stream);
  if (rows == RowType::kBFloat16) return launch_table<__nv_bfloat16>(a, table, vec, stream);
  return launch_table<__half>(a, table, vec, stream);
}

}  // namespace lmc
