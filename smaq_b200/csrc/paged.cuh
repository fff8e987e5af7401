// What the kernels over the exact paged cache share: arguments, score changes, row addresses, and the
// merge of softmax partials.  Scores are kept in the log2 domain: p = 2^(x - m).
#pragma once
#include "common.cuh"
#include "ptx.cuh"

namespace smaq {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct PagedParams {
  smaq_paged_args a;
  int group;             // query heads a KV head
  float scale_log2;      // scale * log2 e: factor of a plain score
  float cap_in;          // capped scores: 2 log2 e * scale / cap, factor inside tanh's exponential
  float cap_log2;        // softcap * log2 e
  float cap_z;           // caps above kCapNear: scale / cap, factor of tanh's argument; 0: others
  FastDiv page_div, group_div;
};

// n / d with a FastDiv of d (0 <= n < 2^31); d == 1 too.
__device__ __forceinline__ int fast_div(int n, const FastDiv& f) {
  return int((uint64_t(__umulhi(uint32_t(n), f.m)) + uint32_t(n)) >> f.l);
}

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// log2-domain score of the product q.k.  Capped: tanh z = 1 - 2 / (e^(2z) + 1), which saturates by itself at both
// ends.  Its absolute error (about 2e-7 here) times the cap is the score's: up to a cap of kCapNear 1.3e-5, a twentieth of
// what rounding a weight to fp16 costs.  Above, scores far below the cap (|z| < 0.3) take the Taylor series of tanh,
// whose first term left out is 5e-8 z, and every score is within 1e-6 of itself.  The series for all caps costs the capped
// decode of 4 x 128K tokens 354 us instead of 337, a branch around it 341, hence CAP_ANY beside CAP_LOW (up to
// kCapNear).  tanh.approx (2^-11) would put 1% errors into the weights at a cap of 30.
constexpr float kCapNear = 64.0f;
enum { CAP_NONE = 0, CAP_LOW = 1, CAP_ANY = 2 };
inline int cap_mode(const smaq_paged_args& a) { return a.softcap > kCapNear ? CAP_ANY : a.softcap > 0.f ? CAP_LOW : CAP_NONE; }
template <int CAP>
__device__ __forceinline__ float score_log2(float qk, const PagedParams& p) {
  if constexpr (CAP != CAP_NONE) {
    float x = fmaf(-2.0f * p.cap_log2, rcp_approx(ex2(qk * p.cap_in) + 1.0f), p.cap_log2);
    if (CAP == CAP_ANY && p.cap_z != 0.f) {  // alike for all
      const float z = qk * p.cap_z, zz = z * z;
      const float near = fmaf(zz, fmaf(zz, fmaf(zz, fmaf(zz, 62.0f / 2835.0f, -17.0f / 315.0f), 2.0f / 15.0f), -1.0f / 3.0f), 1.0f);
      if (fabsf(z) < 0.3f) x = p.cap_log2 * z * near;
    }
    return x;
  } else {
    return qk * p.scale_log2;
  }
}

// Weights are 2^(x - m + kUp): in fp16, whose smallest step is 2^-24, up to 2^15, so that many tokens far below the largest
// still count (at weights of at most 1, those below 2^-25 of it were zero, and 128K of them are 0.4% of an answer).
template <class DT>
constexpr float kUp = DT::code == SMAQ_F16 ? 15.0f : 0.0f;

// Element offset of token j of the request whose table row is `table`, in the K and V caches; the page
// number is clamped to the cache.
__device__ __forceinline__ int64_t token_offset(const PagedParams& p, const int32_t* table, int j) {
  const int blk = fast_div(j, p.page_div);
  const int64_t page = min(max(int64_t(__ldg(table + blk)), int64_t(0)), p.a.n_pages - 1);
  return page * p.a.c_stride_page + int64_t(j - blk * p.a.page_size) * p.a.c_stride_slot;
}

// Length of request b, within its table's width.
constexpr int kLongest = 0x7FFFFF00;
__device__ __forceinline__ int paged_len(const PagedParams& p, int b) {
  const int64_t room = int64_t(p.a.max_blocks) * p.a.page_size;
  const int L = max(__ldg(p.a.seq_lens + b), 0);
  return int(min(min(int64_t(L), room), int64_t(kLongest)));
}

__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
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

// D[16x8] += A[16x16] * B[16x8], fp32 accumulation, both operands of DT.
template <class DT>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (DT::code == SMAQ_F16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// (lo, hi) rounded to DT in one word.
template <class DT>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if constexpr (DT::code == SMAQ_F16) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <class DT>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if constexpr (DT::code == SMAQ_F16) return __half22float2(*reinterpret_cast<__half2*>(&w));
  else return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}

// Checks that both entry points make; p is filled for a launch.
int paged_check(const smaq_paged_args* args, bool prefill, PagedParams& p);
// Whether every row vector of the cache and the queries starts on a 16-byte boundary.
bool paged_aligned(const smaq_paged_args& a);

}  // namespace smaq
