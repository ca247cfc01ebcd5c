// Joins partial results of a row over slices of its keys:
//   o = sum_s 2^(L_s - L) o_s,   L = log2 sum_s 2^L_s
// with o_s normalised in its slice and L_s the base-2 log of its sum.  One warp
// per row, fp32.
#pragma once
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
    join_position_kernel(PositionArgs a, const float *part_o, const float *part_lse, int slices) {
  const long long rows = static_cast<long long>(a.q_tokens) * a.heads;
  const long long row = static_cast<long long>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (row >= rows) return;
  JoinedRow<T, D> r;
  r.join(part_o, part_lse, slices, rows, row);
  if (r.finite())
    r.store(static_cast<T *>(a.out), a.lse, row);
  else
    strict_position_row<T, D>(a, static_cast<int>(row / a.heads), static_cast<int>(row % a.heads));
}

// Score constants of the tensor-core kernel.
inline void set_scores(TcArgs &t, float scale, float softcap) {
  t.scale_log2 = scale * kLog2e;
  t.cap_out = softcap * kLog2e;
  const double u = softcap > 0.f ? static_cast<double>(scale) / softcap : 0.;
  t.cap_in = static_cast<float>(2. * kLog2e * u);
  // tanh(u) / u for |u| <= 0.6 in powers of u^2 (relative minimax by the Remez
  // exchange, degree 4: 7.3e-8), as x / s in powers of s^2.  The powers of a cap
  // that is very wide for its scale leave the fp32 range: it takes the general form.
  constexpr double kRatio[5] = {0.9999999268689601, -0.33332309974406227, 0.13310173658056346,
                                -0.0521014801204608, 0.015475427495065024};
  double f = static_cast<double>(scale) * kLog2e;
  for (int i = 0; i < 5; ++i, f *= u * u)
    t.cap_poly[i].x = t.cap_poly[i].y = static_cast<float>(kRatio[i] * f);
  t.cap_small = u >= 1e-4 ? static_cast<float>(0.6 / u) : -1.f;
}

template <typename T, int D, bool kDense>
cudaError_t launch_tc(const CUtensorMap &k_map, const CUtensorMap &v_map, const TcArgs &t,
                      unsigned grid, cudaStream_t stream) {
  const bool cap = t.cap_out > 0.f, bias = t.slopes != nullptr;
  auto kernel = cap ? (bias ? tc_attention_kernel<T, D, kDense, true, true>
                            : tc_attention_kernel<T, D, kDense, true, false>)
                    : (bias ? tc_attention_kernel<T, D, kDense, false, true>
                            : tc_attention_kernel<T, D, kDense, false, false>);
  constexpr int kBytes = TcSmem<D>::kBytes;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes);
  if (e != cudaSuccess) return e;
  kernel<<<grid, kTcThreads, kBytes, stream>>>(k_map, v_map, t);
  return cudaGetLastError();
}

}  // namespace lmc
