// tcgen05 helpers (sm_100a): descriptors, products from shared and tensor memory, tensor-memory loads and stores.
#pragma once
#include "ptx.cuh"

namespace smaq {
namespace tc5 {

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void alloc(uint32_t* where, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(where)), "r"(cols) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void dealloc(uint32_t tmem, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols) : "memory");
}

// Shared-memory operand in 128-byte swizzled atoms: 8 rows of 128 bytes (64 16-bit elements), 1024 bytes.  `group`: bytes from
// one 8-row group to the next.  K-major: rows are output rows, 64 contraction elements each.  MN-major: rows are
// contraction indices, 64 output elements each, and `next` is the way to the next 64 output elements.
__device__ __forceinline__ uint64_t desc(uint32_t saddr, uint32_t group, uint32_t next) {
  return uint64_t((saddr & 0x3FFFFu) >> 4) | (uint64_t(next >> 4) << 16) | (uint64_t(group >> 4) << 32) | (uint64_t(1) << 46) | (uint64_t(2) << 61);
}
// kind::f16 instruction descriptor: fp32 accumulators, both operands bf16 or fp16, M = 128; B K-major or MN-major.
constexpr uint32_t idesc(bool bf16, uint32_t n, bool b_mn_major) {
  return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (b_mn_major ? 1u << 16 : 0u) | ((n >> 3) << 17) | ((128u >> 4) << 24);
}

// One lane of a converged warp.
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r;
}
// D (tensor memory) (+)= A B^T, A in shared memory / in tensor memory.  The whole warp runs these and only the lane
// with `lead` issues: in code that one lane runs alone, operands live in per-lane registers and every
// product pays for moving them to uniform ones.
__device__ __forceinline__ void mma_ss(uint32_t lead, uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(id), "r"(accumulate), "r"(lead)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t lead, uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(id), "r"(accumulate), "r"(lead)
      : "memory");
}
// Arrives at the barrier when all products that the leading lane issued before are complete.
__device__ __forceinline__ void commit(uint32_t lead, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)),
      "r"(lead)
      : "memory");
}

// 32 columns of this warp's 32 lanes.
__device__ __forceinline__ void ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
        "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]),
      "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]),
      "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Box of a 5-D tensor map to shared memory (no multicast), issued by the lane with `lead`.
__device__ __forceinline__ void tma_5d(uint32_t lead, uint32_t dst, const void* map, int c0, int c1, int c2, int c3, int c4, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %8, 0;\n\t"
      "@q cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];\n\t}" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4), "r"(smem_u32(bar)), "r"(lead)
      : "memory");
}

// 2^x for two x <= 126 on the FMA pipes, whose throughput the special-function unit's exponential lacks: x = n + r
// with n the nearest integer (added to 1.5 2^23 + 127, whose low bits then hold n + 127), 2^n from those bits, 2^r
// by a polynomial with p(0) = 1 of least relative error on [-1/2, 1/2] (fitted by linear programming on
// Chebyshev points): 2.9e-6 for degree 4, 1.9e-7 for 5.  x below -126.5 gives 0 exactly, -infinity
// too; NaN stays NaN.
__device__ constexpr float exp2_coef(int deg, int power) {
  return deg == 4 ? (power == 1 ? 0.6931241750717163f : power == 2 ? 0.24024099111557007f : power == 3 ? 0.055906426161527634f : 0.009582852944731712f)
                  : (power == 1   ? 0.6931470036506653f
                     : power == 2 ? 0.24022242426872253f
                     : power == 3 ? 0.05550733953714371f
                     : power == 4 ? 0.009671511128544807f
                                  : 0.001326465280726552f);
}
// N pairs step by step side by side: one pair alone is a chain of eleven dependent operations.
template <int DEG, int N>
__device__ __forceinline__ void exp2_poly(uint64_t (&x)[N]) {
  constexpr float kMagic = 12582912.0f + 127.0f;
  uint64_t t[N], r[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float2 v = split(x[i]);
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(v.x) : "f"(-127.0f));
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(v.y) : "f"(-127.0f));
    x[i] = pair(v.x, v.y);
  }
#pragma unroll
  for (int i = 0; i < N; ++i) t[i] = add2(x[i], pair(kMagic, kMagic));
#pragma unroll
  for (int i = 0; i < N; ++i) r[i] = add2(t[i], pair(-kMagic, -kMagic));
#pragma unroll
  for (int i = 0; i < N; ++i) r[i] = fma2(r[i], pair(-1.0f, -1.0f), x[i]);
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = fma2(pair(exp2_coef(DEG, DEG), exp2_coef(DEG, DEG)), r[i], pair(exp2_coef(DEG, DEG - 1), exp2_coef(DEG, DEG - 1)));
#pragma unroll
  for (int d = DEG - 2; d >= 1; --d)
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = fma2(x[i], r[i], pair(exp2_coef(DEG, d), exp2_coef(DEG, d)));
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = fma2(x[i], r[i], pair(1.0f, 1.0f));
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float2 n = split(t[i]);
    x[i] = mul2(x[i], pair(__uint_as_float(__float_as_uint(n.x) << 23), __uint_as_float(__float_as_uint(n.y) << 23)));
  }
}

}  // namespace tc5
}  // namespace smaq
