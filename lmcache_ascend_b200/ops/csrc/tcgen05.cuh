// Blackwell tensor-core building blocks: tensor memory, tcgen05.mma and its
// descriptors, tiled TMA loads (never multicast), and waits that end.
#pragma once
#include <cuda.h>

#include "common.cuh"

namespace lmc {

// --- tensor memory (one warp allocates and frees; 512 columns = the SM's whole)
__device__ __forceinline__ void tmem_alloc(uint32_t *smem_dst, uint32_t columns) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                   smem_u32(smem_dst)),
               "r"(columns)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void tmem_free(uint32_t addr, uint32_t columns) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(columns));
}

__device__ __forceinline__ void tc_fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tmem_wait_ld() {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_wait_st() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// 32 columns of the warp's 32 lanes: register i of a thread is column i of its lane.
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}

// One lane of a converged warp.  Descriptors of tcgen05.mma live in uniform
// registers: under this predicate, with operands that are the same in the whole
// warp, the compiler keeps them there (under `lane == 0` it moves each one over,
// and the mma waited on those moves half the time).
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile(
      "{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}"
      : "=r"(r));
  return r != 0;
}

__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// --- tcgen05.mma, kind::f16, fp32 accumulators, one CTA
// Instruction descriptor: D fp32, A and B of one 16-bit type (bf16 or f16), A
// K-major, B K-major or (b_mn) MN-major, M x N.
__device__ __forceinline__ constexpr uint32_t mma_desc(bool bf16, bool b_mn, int m, int n) {
  return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) |
         ((b_mn ? 1u : 0u) << 16) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(m >> 4) << 24);
}

// Shared-memory operand in 128-byte swizzled rows: 8-row groups `sbo` bytes
// apart; for an MN-major operand 64-element column blocks `lbo` bytes apart.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
  return static_cast<uint64_t>((addr & 0x3ffff) >> 4) | (static_cast<uint64_t>(lbo >> 4) << 16) |
         (static_cast<uint64_t>(sbo >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                       bool accumulate) {
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.u32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate ? 1u : 0u)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                       bool accumulate) {
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.u32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate ? 1u : 0u)
      : "memory");
}

// The barrier gets one arrival when all earlier mma of this thread are done.
__device__ __forceinline__ void mma_commit(uint64_t *bar) {
  asm volatile(
      "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
          smem_u32(bar))
      : "memory");
}

// --- tiled TMA loads of this GPU's own memory
__device__ __forceinline__ void prefetch_map(const CUtensorMap *map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}
__device__ __forceinline__ void tma_load_3d(void *dst, const CUtensorMap *map, int x, int y, int z,
                                            uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(dst)),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void tma_load_4d(void *dst, const CUtensorMap *map, int x, int y, int z,
                                            int w, uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(smem_u32(dst)),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
      : "memory");
}

__device__ __forceinline__ void mbar_arrive(uint64_t *bar) {
  asm volatile("mbarrier.arrive.release.cta.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar))
               : "memory");
}

// Up to 2^16 tries for a phase, of at most about a microsecond each.  The loop is
// in one asm block: written around the try in C++ the way out of it cost 300
// cycles per wait, also when the phase was long complete.
__device__ __forceinline__ bool tries(uint64_t *bar, unsigned parity) {
  uint32_t done;
  asm volatile(
      "{\n.reg .pred p, q;\n.reg .u32 n;\nmov.u32 n, 0;\n"
      "again_%=:\n"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, 1000;\n"
      "@p bra done_%=;\n"
      "add.u32 n, n, 1;\nsetp.lt.u32 q, n, 65536;\n@q bra again_%=;\n"
      "done_%=:\nselp.u32 %0, 1, 0, p;\n}"
      : "=r"(done)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return done != 0;
}

__device__ __forceinline__ bool phase_done(uint64_t *bar, unsigned parity) {
  uint32_t done;
  asm volatile(
      "{\n.reg .pred p;\nmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n"
      "selp.u32 %0, 1, 0, p;\n}"
      : "=r"(done)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return done != 0;
}

// One lane's wait; see wait_or_stop.  At most 32 x 2^16 tries.
__device__ __forceinline__ bool lane_wait(uint64_t *bar, unsigned parity, int *stopped) {
  if (phase_done(bar, parity)) return true;  // a third of the time of a try
  if (__builtin_expect(tries(bar, parity), 1)) return true;
#pragma unroll 1
  for (int i = 0; i < 31; ++i) {
    if (*reinterpret_cast<volatile int *>(stopped)) return false;
    if (tries(bar, parity)) return true;
  }
  *reinterpret_cast<volatile int *>(stopped) = 1;
  return false;
}

// A whole warp's wait for a phase, with an end: after some two million tries (0.1
// to 2 seconds), or soon after another warp of the block gave up, the block's
// flag is set and every lane of the caller gets false.
__device__ __forceinline__ bool wait_or_stop(uint64_t *bar, unsigned parity, int *stopped) {
  return __all_sync(0xffffffffu, lane_wait(bar, parity, stopped));
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// --- pairs of fp32 in one instruction
using f32x2 = unsigned long long;
__device__ __forceinline__ f32x2 pack2(float a, float b) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(f32x2 v, float &a, float &b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// 2^x for x below 128 on the FMA pipe: x = j + f with f in [-1/2, 1/2], a
// degree-5 polynomial for 2^f (relative minimax over the interval by the Remez
// exchange: 7.5e-8, 2.3e-7 in fp32 Horner form, as exact as ex2) and j added to
// the exponent.  Below 2^-126 it stays there (weights of that size vanish next
// to the row's largest); NaN and what it leads to stay outside the finite range.
__device__ __forceinline__ void exp2_fma(f32x2 x, float &a, float &b) {
  constexpr float kShift = 12582912.f;  // 1.5 * 2^23: adding it rounds to an integer
  unpack2(x, a, b);
  x = pack2(max_nan(a, -126.f), max_nan(b, -126.f));
  const f32x2 t = add2(x, pack2(kShift, kShift));
  const f32x2 f = fma2(add2(t, pack2(-kShift, -kShift)), pack2(-1.f, -1.f), x);
  f32x2 p = pack2(0.0013276472454890609f, 0.0013276472454890609f);
  p = fma2(p, f, pack2(0.009675540961325169f, 0.009675540961325169f));
  p = fma2(p, f, pack2(0.05550713092088699f, 0.05550713092088699f));
  p = fma2(p, f, pack2(0.24022120237350464f, 0.24022120237350464f));
  p = fma2(p, f, pack2(0.6931469440460205f, 0.6931469440460205f));
  p = fma2(p, f, pack2(1.0000001192092896f, 1.0000001192092896f));
  float ta, tb;
  unpack2(t, ta, tb);
  unpack2(p, a, b);
  a = __uint_as_float(__float_as_uint(a) + (__float_as_uint(ta) << 23));
  b = __uint_as_float(__float_as_uint(b) + (__float_as_uint(tb) << 23));
}

}  // namespace lmc
