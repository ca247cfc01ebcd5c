// What the attention kernels share: their arguments, the score, and the row
// that one warp computes by the definition.
//
// For a query row and the keys it sees
//   x_j = scale * q . k_j,   x_j = cap * tanh(x_j / cap)      (cap > 0)
//   x_j = x_j - slope_h * |p - p_j|                            (distance bias)
//   o = sum_j exp(x_j - lse) v_j,   lse = log sum_j exp(x_j)
// with every sum and statistic in fp32 and one rounding of o to the row's type.
// A row that sees no key is zero with lse = -inf; one whose scores are all -inf has
// no weights and is NaN.  Keys it does not see are
// never multiplied by a zero weight: whatever their rows hold stays out.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "common.cuh"
#include "serving_ops.h"

namespace lmc {

static_assert(sizeof(DeviceStatus) == kDeviceStatusBytes, "status layout");

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

template <typename T>
__device__ __forceinline__ float2 pair_to_float(uint32_t w);
template <>
__device__ __forceinline__ float2 pair_to_float<__nv_bfloat16>(uint32_t w) {
  return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162 *>(&w));
}
template <>
__device__ __forceinline__ float2 pair_to_float<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<__half2 *>(&w));
}
template <typename T>
__device__ __forceinline__ uint32_t pair_from_float(float a, float b);
template <>
__device__ __forceinline__ uint32_t pair_from_float<__nv_bfloat16>(float a, float b) {
  __nv_bfloat162 w = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t *>(&w);
}
template <>
__device__ __forceinline__ uint32_t pair_from_float<__half>(float a, float b) {
  __half2 w = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t *>(&w);
}

// --- 16-byte asynchronous copies; with `valid` false zeros, nothing is read
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(valid ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// --- overlapped launches of one call (see launch_ordered)
__device__ __forceinline__ void let_next_start() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
__device__ __forceinline__ void wait_for_previous() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// One query row on one warp, 32 keys at a time: lane i multiplies key i with the
// query, then the lanes go over the values together, lane l for the row's elements
// [l D/32, (l + 1) D/32).  For rows that are computed a second time; where most rows
// of a call see an infinity it is this loop that sets the time (4096 rows of 32/8
// heads of 128, causal, an infinity in every head's first value: 29 ms against 0.4
// without; 148 a key at a time).
template <typename T, int D>
struct WarpRow {
  static constexpr int E = D / 32;
  const T *q;
  float o[E], m, l;
  bool lowest;  // there was a score of -inf before any other

  __device__ __forceinline__ void start(const T *row) {
    q = row;
#pragma unroll
    for (int i = 0; i < E; ++i) o[i] = 0.f;
    m = -INFINITY;
    l = 0.f;
    lowest = false;
  }

  // Once a weight is NaN so is all of the row: no key changes it.
  __device__ __forceinline__ bool lost() const { return l != l; }

  // This lane's key and value (`sees` false: none); bias is subtracted after the cap.
  __device__ __forceinline__ void add(bool sees, const T *k, const T *v, float scale, float cap,
                                      float bias) {
    constexpr uint32_t kAll = 0xffffffffu;
    const uint32_t seen = __ballot_sync(kAll, sees);
    if (seen == 0) return;
    float x = 0.f;
    if (sees) {
#pragma unroll 4
      for (int c = 0; c < D / 8; ++c) {
        const uint4 a = reinterpret_cast<const uint4 *>(q)[c];
        const uint4 b = reinterpret_cast<const uint4 *>(k)[c];
        const uint32_t *aw = &a.x, *bw = &b.x;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 f = pair_to_float<T>(aw[i]), g = pair_to_float<T>(bw[i]);
          x = fmaf(f.x, g.x, x);
          x = fmaf(f.y, g.y, x);
        }
      }
      x *= scale;
      if (cap > 0.f) x = cap * tanhf(x / cap);
      x = (x - bias) * kLog2e;
    }
    float top = sees ? x : -INFINITY;  // (a NaN score leaves the maximum)
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) top = fmaxf(top, __shfl_xor_sync(kAll, top, s));
    top = fmaxf(m, top);
    if (top == -INFINITY) {  // scores of -inf or NaN, before any other
      lowest = true;
      if (__any_sync(kAll, sees && x != x)) l = NAN;
      return;
    }
    const float keep = exp2f(m - top), w = sees ? exp2f(x - top) : 0.f;
    m = top;
    float sum = w;
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) sum += __shfl_xor_sync(kAll, sum, s);
    l = l * keep + sum;
#pragma unroll
    for (int i = 0; i < E; ++i) o[i] *= keep;
    // a key that is not seen has a place that can be read, and its value stays out
    const auto at = reinterpret_cast<unsigned long long>(v);
    const unsigned long long first = __shfl_sync(kAll, at, __ffs(seen) - 1);
    const unsigned long long mine = sees ? at : first;
    const int e0 = (threadIdx.x & 31) * E;
#pragma unroll 8
    for (int b = 0; b < 32; ++b) {
      const T *row = reinterpret_cast<const T *>(__shfl_sync(kAll, mine, b)) + e0;
      const float wb = __shfl_sync(kAll, w, b);
      const bool in = (seen >> b) & 1;
#pragma unroll
      for (int i = 0; i < E / 2; ++i) {
        const float2 f = pair_to_float<T>(reinterpret_cast<const uint32_t *>(row)[i]);
        o[2 * i] = fmaf(wb, in ? f.x : 0.f, o[2 * i]);
        o[2 * i + 1] = fmaf(wb, in ? f.y : 0.f, o[2 * i + 1]);
      }
    }
  }

  __device__ __forceinline__ void finish(T *row, float *lse) const {
    // scores of -inf only have no weights: NaN
    const float inv = l == 0.f ? (lowest ? NAN : 0.f) : 1.f / l;
    uint32_t *w = reinterpret_cast<uint32_t *>(row + (threadIdx.x & 31) * E);
#pragma unroll
    for (int i = 0; i < E / 2; ++i)
      w[i] = pair_from_float<T>(o[2 * i] * inv, o[2 * i + 1] * inv);
    if (lse != nullptr && (threadIdx.x & 31) == 0)
      *lse = l == 0.f ? (lowest ? NAN : -INFINITY) : m * kLn2 + logf(l);
  }
};

__device__ __forceinline__ long long position_at(const void *p, bool is_long, int i) {
  return is_long ? static_cast<const long long *>(p)[i]
                 : static_cast<long long>(static_cast<const int *>(p)[i]);
}

}  // namespace lmc
