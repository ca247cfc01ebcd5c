// Joins partial results of a row over slices of its keys:
//   o = sum_s 2^(L_s - L) o_s,   L = log2 sum_s 2^L_s
// with o_s normalised in its slice and L_s the base-2 log of its sum.  One warp
// per row, fp32.
#pragma once
#include <algorithm>
#include <mutex>
#include <set>
#include <utility>

#include "tc_attention.cuh"

namespace lmc {

template <typename T, int D>
struct JoinedRow {
  static constexpr int E = D / 32;
  float o[E], log2_sum;

  __device__ __forceinline__ void join(const float *part_o, const float *part_lse, int slices,
                                       long long rows, long long row) {
    const int lane = threadIdx.x & 31;
    float top = -INFINITY;
    for (int s = lane; s < slices; s += 32) top = fmaxf(top, part_lse[s * rows + row]);
#pragma unroll
    for (int i = 16; i > 0; i >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, i));
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) o[i] = 0.f;
    const float off = top == -INFINITY ? 0.f : top;
    for (int s = 0; s < slices; ++s) {
      const float part = part_lse[s * rows + row];
      if (part == -INFINITY) continue;  // an empty slice (its o is not read)
      const float w = exp2f(part - off);
      sum += w;
      const float *p = part_o + (s * rows + row) * D + lane * E;
#pragma unroll
      for (int i = 0; i < E; i += 2) {
        const float2 v = *reinterpret_cast<const float2 *>(p + i);
        o[i] = fmaf(w, v.x, o[i]);
        o[i + 1] = fmaf(w, v.y, o[i + 1]);
      }
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int i = 0; i < E; ++i) o[i] *= inv;
    log2_sum = sum == 0.f ? -INFINITY : off + log2f(sum);
  }

  __device__ __forceinline__ bool finite() const {
    bool ok = true;
#pragma unroll
    for (int i = 0; i < E; ++i) ok = ok && fabsf(o[i]) <= 3.4028235e38f;
    return __all_sync(0xffffffffu, ok && !(log2_sum > 3.4028235e38f));
  }

  __device__ __forceinline__ void store(T *out, float *lse, long long row) const {
    const int lane = threadIdx.x & 31;
    uint32_t *w = reinterpret_cast<uint32_t *>(out + row * D + lane * E);
#pragma unroll
    for (int i = 0; i < E / 2; ++i) w[i] = pair_from_float<T>(o[2 * i], o[2 * i + 1]);
    if (lse != nullptr && lane == 0) lse[row] = log2_sum * kLn2;
  }
};

template <typename T, int D>
__global__ void __launch_bounds__(128)
    join_position_kernel(const __grid_constant__ PositionArgs a, const float *part_o,
                         const float *part_lse, int slices) {
  const long long rows = static_cast<long long>(a.q_tokens) * a.heads;
  const long long row = static_cast<long long>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  wait_for_previous();
  if (row >= rows) return;
  JoinedRow<T, D> r;
  r.join(part_o, part_lse, slices, rows, row);
  if (r.finite())
    r.store(static_cast<T *>(a.out), a.lse, row);
  else
    strict_position_row_again<T, D>(a, static_cast<int>(row / a.heads),
                                    static_cast<int>(row % a.heads));
}

// Score constants of the tensor-core kernel.
inline void set_scores(TcArgs &t, float scale, float softcap) {
  t.scale_log2 = scale * kLog2e;
  t.cap_out = softcap * kLog2e;
  const double u = softcap > 0.f ? static_cast<double>(scale) / softcap : 0.;
  t.cap_u = static_cast<float>(u);
  t.cap_in = static_cast<float>(2. * kLog2e * u);
  // tanh(u) / u for |u| <= 0.6 in powers of u^2 (relative minimax by the Remez
  // exchange, degree 4: 7.3e-8), times the score's scale
  constexpr double kRatio[5] = {0.9999999268689601, -0.33332309974406227, 0.13310173658056346,
                                -0.0521014801204608, 0.015475427495065024};
  for (int i = 0; i < 5; ++i)
    t.cap_poly[i].x = t.cap_poly[i].y = static_cast<float>(kRatio[i] * scale * kLog2e);
  t.cap_small = static_cast<float>(0.6 / std::max(u, 1e-37));
}

// Lets a kernel use `bytes` of shared memory on the current device; asked of the
// runtime once per device (the call costs as much as a launch).
template <typename Kernel>
cudaError_t allow_smem(Kernel kernel, int bytes) {
  static std::mutex lock;
  static std::set<std::pair<const void *, int>> done;
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  const std::lock_guard<std::mutex> hold(lock);
  const auto key = std::make_pair(reinterpret_cast<const void *>(kernel), device);
  if (done.count(key)) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done.insert(key);
  return e;
}

// Launches one of a call's kernels.  The first waits for all that was in the
// stream before it; the blocks of a later one may start while the kernel before
// it ends (it hides the launch and fills the SMs that are done).  Every kernel
// calls wait_for_previous() before it reads what an earlier one of the call
// wrote, and in any case before its blocks end, so that they complete in order.
// `cluster`: blocks of a cluster along y.
template <typename... Params, typename... Args>
cudaError_t launch_ordered(void (*kernel)(Params...), dim3 grid, unsigned threads, int smem,
                           bool first, cudaStream_t stream, int cluster, const Args &...args) {
  cudaLaunchConfig_t config = {};
  config.gridDim = grid;
  config.blockDim = dim3(threads);
  config.dynamicSmemBytes = static_cast<size_t>(smem);
  config.stream = stream;
  cudaLaunchAttribute attributes[2] = {};
  config.attrs = attributes;
  if (!first) {
    attributes[config.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[config.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 1) {
    attributes[config.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attributes[config.numAttrs++].val.clusterDim = {1, static_cast<unsigned>(cluster), 1};
  }
  return cudaLaunchKernelEx(&config, kernel, Params(args)...);
}

template <typename T, int D, bool kDense, bool kDocs>
cudaError_t launch_tc(const CUtensorMap &k_map, const CUtensorMap &v_map, const TcArgs &t,
                      unsigned grid, bool first, cudaStream_t stream) {
  const bool cap = t.cap_out > 0.f, bias = t.slopes != nullptr;
  auto kernel = cap ? (bias ? tc_attention_kernel<T, D, kDense, kDocs, true, true>
                            : tc_attention_kernel<T, D, kDense, kDocs, true, false>)
                    : (bias ? tc_attention_kernel<T, D, kDense, kDocs, false, true>
                            : tc_attention_kernel<T, D, kDense, kDocs, false, false>);
  constexpr int kBytes = TcSmem<D>::kBytes;
  cudaError_t e = allow_smem(kernel, kBytes);
  if (e != cudaSuccess) return e;
  return launch_ordered(kernel, dim3(grid), kTcThreads, kBytes, first, stream, 1, k_map, v_map, t);
}

}  // namespace lmc
