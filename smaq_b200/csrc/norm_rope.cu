// Per-head RMS norm and rotation of queries and keys, with the cache write of keys and values, in one
// pass: every row is read once and written once, 32-bit arithmetic in between, one rounding.
//
//   y = x / sqrt(mean x^2 + eps) * w;   (a, b) -> (a cos - b sin, b cos + a sin)
//
// norm_rope_kernel: a head is held by head_dim / 16 lanes (padded to a power of two), two 8-element
// vectors a lane.  A lane of the rotated part holds elements [8l, 8l + 8) and the same of the second
// half, so both partners of every pair, (i, i + R/2) as well as (2i, 2i + 1), are in one lane and the
// rotation needs no exchange; only the sum of squares crosses lanes.  The cosines and sines of a token
// are read once into registers and serve all heads that the lane group walks; it walks more heads a token
// when there are enough tokens to fill the GPU, and loads a head ahead.  Values are copied by the same
// walk.  Bound by latency: of a launch for decode steps, of loads and dependent arithmetic for prompts.
// norm_rope_staged_kernel: the same arithmetic for many tokens, rows staged in shared memory by bulk copies.
// norm_rope_any_kernel: any head_dim and alignment, one warp a head, element by element.
#include "common.cuh"
#include "ptx.cuh"

namespace smaq {

namespace {

struct NrParams {
  smaq_norm_rope_args a;
  int heads;            // q + k (+ v with a cache)
  uint32_t spin;        // polls before a wait gives up
  int per;              // heads that a lane group walks
  int groups, q_groups, k_groups;  // lane groups a token, of its queries and of its keys (and values)
  float inv_dim;
  FastDiv page_div;
};

constexpr int NR_THREADS = 128;
constexpr int NR_CTAS = 6;  // an SM: 80 registers; 64 spill (67 us), 104 hold too few loads in flight (78 us)
constexpr int NR_PER = 2;   // heads a lane group walks at most: 1, 2, 4, 8, 16 took 91, 54, 56, 62, 70 us at 8192 tokens

// Element offset of slot `s` in the cache, < 0 for one outside it.
__device__ __forceinline__ int64_t slot_offset(const NrParams& p, int64_t s) {
  const smaq_norm_rope_args& a = p.a;
  if (s < 0 || s >= a.n_pages * a.page_size) return -1;
  int64_t page;
  if (s < (int64_t(1) << 31)) page = int64_t((uint64_t(__umulhi(uint32_t(s), p.page_div.m)) + uint32_t(s)) >> p.page_div.l);
  else page = s / a.page_size;
  return page * a.c_stride_page + (s - page * a.page_size) * a.c_stride_slot;
}

template <class DT>
struct Vec8;  // eight elements
template <>
struct Vec8<BF16> {
  uint4 u;
};
template <>
struct Vec8<F16> {
  uint4 u;
};
template <>
struct Vec8<F32> {
  float4 u, w;
};

template <class DT>
__device__ __forceinline__ Vec8<DT> load8(const typename DT::T* p) {
  Vec8<DT> v;
  v.u = __ldg(reinterpret_cast<const decltype(v.u)*>(p));
  if constexpr (DT::code == SMAQ_F32) v.w = __ldg(reinterpret_cast<const float4*>(p) + 1);
  return v;
}
template <class DT>
__device__ __forceinline__ Vec8<DT> load8s(const typename DT::T* p) {  // from shared memory
  Vec8<DT> v;
  v.u = *reinterpret_cast<const decltype(v.u)*>(p);
  if constexpr (DT::code == SMAQ_F32) v.w = reinterpret_cast<const float4*>(p)[1];
  return v;
}
template <class DT>
__device__ __forceinline__ void store8(typename DT::T* p, const Vec8<DT>& v) {
  *reinterpret_cast<decltype(v.u)*>(p) = v.u;
  if constexpr (DT::code == SMAQ_F32) reinterpret_cast<float4*>(p)[1] = v.w;
}
// Eight elements as four packed pairs of 32-bit values.
template <class DT>
__device__ __forceinline__ void unpack8(const Vec8<DT>& v, uint64_t* x) {
  if constexpr (DT::code == SMAQ_F32) {
    x[0] = pair(v.u.x, v.u.y);
    x[1] = pair(v.u.z, v.u.w);
    x[2] = pair(v.w.x, v.w.y);
    x[3] = pair(v.w.z, v.w.w);
  } else {
    const uint32_t w[4] = {v.u.x, v.u.y, v.u.z, v.u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT::code == SMAQ_BF16) {
        x[i] = pair(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u));
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        x[i] = pair(f.x, f.y);
      }
    }
  }
}
template <class DT>
__device__ __forceinline__ Vec8<DT> pack8(const uint64_t* x) {
  Vec8<DT> v;
  const float2 f0 = split(x[0]), f1 = split(x[1]), f2 = split(x[2]), f3 = split(x[3]);
  if constexpr (DT::code == SMAQ_F32) {
    v.u = make_float4(f0.x, f0.y, f1.x, f1.y);
    v.w = make_float4(f2.x, f2.y, f3.x, f3.y);
  } else if constexpr (DT::code == SMAQ_BF16) {
    auto two = [](float2 f) { uint32_t r; asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(f.y), "f"(f.x)); return r; };
    v.u = make_uint4(two(f0), two(f1), two(f2), two(f3));
  } else {
    v.u = make_uint4(pack_f16x2(f0.x, f0.y), pack_f16x2(f1.x, f1.y), pack_f16x2(f2.x, f2.y), pack_f16x2(f3.x, f3.y));
  }
  return v;
}
__device__ __forceinline__ void load8f(const float* p, uint64_t* x) {
  const float4 u = __ldg(reinterpret_cast<const float4*>(p)), w = __ldg(reinterpret_cast<const float4*>(p) + 1);
  x[0] = pair(u.x, u.y);
  x[1] = pair(u.z, u.w);
  x[2] = pair(w.x, w.y);
  x[3] = pair(w.z, w.w);
}

// Turns this lane's eight pairs.  Interleaved: the cosines and sines of vector a's four pairs, then b's.
template <bool INTERLEAVED>
__device__ __forceinline__ void rotate(uint64_t (&x)[8], const uint64_t (&c)[4], const uint64_t (&s)[4]) {
  if constexpr (INTERLEAVED) {  // a packed pair is a rotated pair
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 u = split(x[i]), c2 = split(c[i >> 1]), s2 = split(s[i >> 1]);
      const float cc = i & 1 ? c2.y : c2.x, sn = i & 1 ? s2.y : s2.x;
      x[i] = pair(u.x * cc - u.y * sn, u.y * cc + u.x * sn);
    }
  } else {  // pair i is (i, i + 8) of this lane's sixteen
    const uint64_t minus = pair(-1.0f, -1.0f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint64_t u = x[i], v = x[i + 4];
      x[i] = fma2(mul2(v, s[i]), minus, mul2(u, c[i]));
      x[i + 4] = fma2(v, c[i], mul2(u, s[i]));
    }
  }
}

// LANES lanes a head (a power of two >= head_dim / 16).  A lane group walks `per` heads of one kind (queries, keys
// or values) of one token.
template <class DT, int LANES, bool INTERLEAVED>
__global__ void __launch_bounds__(NR_THREADS, NR_CTAS) norm_rope_kernel(const __grid_constant__ NrParams p) {
  using T = typename DT::T;
  const smaq_norm_rope_args& a = p.a;
  const int lane = threadIdx.x % LANES;
  const int64_t job = int64_t(blockIdx.x) * (NR_THREADS / LANES) + threadIdx.x / LANES;
  const int64_t t = job / p.groups;
  if (t >= a.n_tokens) return;  // whole lane groups leave; the shuffles below name the group's lanes
  const unsigned mask = (LANES == 32 ? ~0u : ((1u << LANES) - 1u) << ((threadIdx.x & 31) / LANES * LANES));
  const int D = a.head_dim, R = a.rotary_dim;
  int g = int(job - t * p.groups), kind = 0;
  if (g >= p.q_groups) {
    g -= p.q_groups;
    kind = 1 + (g >= p.k_groups);
    if (kind == 2) g -= p.k_groups;
  }
  const int h0 = g * p.per;
  int left = min(p.per, (kind ? a.n_kv_heads : a.n_q_heads) - h0);
  const bool live = lane < D / 16, turned = lane < R / 16;
  // this lane's two vectors
  const int ea = turned ? 8 * lane : R + 16 * (lane - R / 16), ahead = turned ? R / 2 : 8;

  const int64_t in_step = kind == 0 ? a.q_stride_h : kind == 1 ? a.k_stride_h : a.v_stride_h;
  const T* src = static_cast<const T*>(kind == 0 ? a.q : kind == 1 ? a.k : a.v) +
                 t * (kind == 0 ? a.q_stride_t : kind == 1 ? a.k_stride_t : a.v_stride_t) + h0 * in_step + ea;
  T *dst, *also = nullptr;  // also: keys may go to the cache and to k_out
  int64_t step = D;
  if (kind == 0) {
    dst = static_cast<T*>(a.q_out) + (t * a.n_q_heads + h0) * D + ea;
  } else {
    if (kind == 1 && a.k_out) also = static_cast<T*>(a.k_out) + (t * a.n_kv_heads + h0) * D + ea;
    const int64_t at = a.k_cache ? slot_offset(p, a.slots[t]) : -1;
    dst = at < 0 ? nullptr : static_cast<T*>(kind == 1 ? a.k_cache : a.v_cache) + at + h0 * a.c_stride_h + ea;
    step = a.c_stride_h;
  }
  Vec8<DT> na = {}, nb = {};  // the next head's
  if (live) {
    na = load8<DT>(src);
    nb = load8<DT>(src + ahead);
  }
  if (kind == 2) {
    while (left-- > 0) {
      const Vec8<DT> va = na, vb = nb;
      if (!live) continue;
      if (left > 0) {
        src += in_step;
        na = load8<DT>(src);
        nb = load8<DT>(src + ahead);
      }
      if (dst) {
        store8<DT>(dst, va);
        store8<DT>(dst + ahead, vb);
        dst += step;
      }
    }
    return;
  }
  uint64_t c[4], s[4], w[8];  // interleaved: the cosines and sines of vector a's four pairs, then b's
  if (turned) {
    const int pos = a.positions[t];
    if (pos >= 0 && pos < a.n_positions) {
      const float* row = a.table + int64_t(pos) * R;
      if constexpr (INTERLEAVED) {  // pair i of either vector is pair (its first element) / 2 + i
        const float4 ca = __ldg(reinterpret_cast<const float4*>(row + ea / 2)), cb = __ldg(reinterpret_cast<const float4*>(row + (ea + ahead) / 2));
        row += R / 2;
        const float4 sa = __ldg(reinterpret_cast<const float4*>(row + ea / 2)), sb = __ldg(reinterpret_cast<const float4*>(row + (ea + ahead) / 2));
        c[0] = pair(ca.x, ca.y); c[1] = pair(ca.z, ca.w); c[2] = pair(cb.x, cb.y); c[3] = pair(cb.z, cb.w);
        s[0] = pair(sa.x, sa.y); s[1] = pair(sa.z, sa.w); s[2] = pair(sb.x, sb.y); s[3] = pair(sb.z, sb.w);
      } else {
        load8f(row + ea, c);
        load8f(row + R / 2 + ea, s);
      }
    } else {
      const float nan = __int_as_float(0x7FC00000);
#pragma unroll
      for (int i = 0; i < 4; ++i) c[i] = s[i] = pair(nan, nan);
    }
  }
  const float* weight = kind ? a.k_weight : a.q_weight;
  if (weight && live) {
    load8f(weight + ea, w);
    load8f(weight + ea + ahead, w + 4);
  }
  while (left-- > 0) {
    uint64_t x[8];
    unpack8<DT>(na, x);
    unpack8<DT>(nb, x + 4);
    if (left > 0 && live) {
      src += in_step;
      na = load8<DT>(src);
      nb = load8<DT>(src + ahead);
    }
    if (weight) {
      uint64_t sq[2] = {0, 0};
      if (live) {
#pragma unroll
        for (int i = 0; i < 8; ++i) sq[i & 1] = fma2(x[i], x[i], sq[i & 1]);
      }
      const float2 f = split(add2(sq[0], sq[1]));
      float ss = f.x + f.y;
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(mask, ss, o);
      const float r = rsqrtf(fmaf(ss, p.inv_dim, a.eps));
      const uint64_t r2 = pair(r, r);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = mul2(x[i], mul2(r2, w[i]));
    }
    if (turned) rotate<INTERLEAVED>(x, c, s);
    if (!live) continue;
    const Vec8<DT> va = pack8<DT>(x), vb = pack8<DT>(x + 4);
    if (dst) {
      store8<DT>(dst, va);
      store8<DT>(dst + ahead, vb);
      dst += step;
    }
    if (also) {
      store8<DT>(also, va);
      store8<DT>(also + ahead, vb);
      also += D;
    }
  }
}

// ---------------------------------------------------------------- many tokens
// The rows of `per` tokens at a time come to shared memory by bulk copies, two batches in turn, so that bytes in
// flight do not cost registers; a lane group then takes head after head of one token from there (8192 tokens at 32/8 heads:
// 45.5 us, 4.5 TB/s; an elementwise pass over as many bytes takes 33).  Values go from shared memory
// to the cache by bulk copies too.  For heads that lie side by side in a token.  Sixteen warps an SM issue in 41% of the
// cycles; the others go to the barrier between batches, to loads, and to results that the next instruction waits for.
constexpr int NS_THREADS = 256, NS_CTAS = 2, NS_SMEM = 112 * 1024, NS_MOST = 16;
constexpr int NS_ROUNDS = 3;

__device__ unsigned int g_norm_rope_fault;

__device__ __forceinline__ void bulk_s2g(void* dst, uint32_t src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(src), "r"(bytes) : "memory");
}

struct NsBars {
  uint64_t full[2];
  int dead;             // a wait ran out
  int pos[2][NS_MOST];  // table rows of a batch's tokens, < 0: outside the table
};

template <class DT, int LANES, bool INTERLEAVED>
__global__ void __launch_bounds__(NS_THREADS, NS_CTAS) norm_rope_staged_kernel(const __grid_constant__ NrParams p) {
  using T = typename DT::T;
  constexpr int GROUPS = NS_THREADS / LANES;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ NsBars bars;
  const smaq_norm_rope_args& a = p.a;
  const int D = a.head_dim, R = a.rotary_dim, lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
  const unsigned mask = (LANES == 32 ? ~0u : ((1u << LANES) - 1u) << ((threadIdx.x & 31) / LANES * LANES));
  const uint32_t row = uint32_t(D * sizeof(T)), q_bytes = a.n_q_heads * row, k_bytes = a.n_kv_heads * row, r_bytes = R * 4;
  const uint32_t v_bytes = a.k_cache ? k_bytes : 0, token = q_bytes + k_bytes + v_bytes + r_bytes, batch = token * p.per;
  const bool live = lane < D / 16, turned = lane < R / 16;
  const int ea = turned ? 8 * lane : R + 16 * (lane - R / 16), ahead = turned ? R / 2 : 8;
  const int64_t batches = (a.n_tokens + p.per - 1) / p.per;
  // A lane group serves one token of a batch: heads first, first + share, ..; its cosines and weights stay in registers.
  const int share = GROUPS / p.per, mine = group / share, first = group - mine * share;
  uint64_t wq[8] = {}, wk[8] = {};
  if (live && a.q_weight) {
    load8f(a.q_weight + ea, wq);
    load8f(a.q_weight + ea + ahead, wq + 4);
  }
  if (live && a.k_weight) {
    load8f(a.k_weight + ea, wk);
    load8f(a.k_weight + ea + ahead, wk + 4);
  }

  // the first warp brings a batch: lane i its token i
  auto bring = [&](int64_t n, int s) {
    const int64_t t = n * p.per + threadIdx.x;
    const bool has = int(threadIdx.x) < p.per && t < a.n_tokens;
    const int pos = has ? a.positions[t] : -1;
    const bool known = pos >= 0 && pos < a.n_positions;
    if (has) bars.pos[s][threadIdx.x] = known ? pos : -1;
    const uint32_t bytes = has ? token - (known ? 0 : r_bytes) : 0;
    const uint32_t total = __reduce_add_sync(~0u, bytes);
    __syncwarp();  // the positions are written before the arrival that publishes them
    if (threadIdx.x == 0) mbar_arrive_expect_tx(&bars.full[s], total);
    __syncwarp();
    if (!has) return;
    uint8_t* dst = smem + s * batch + threadIdx.x * token;
    bulk_g2s(dst, static_cast<const T*>(a.q) + t * a.q_stride_t, q_bytes, &bars.full[s]);
    bulk_g2s(dst + q_bytes, static_cast<const T*>(a.k) + t * a.k_stride_t, k_bytes, &bars.full[s]);
    if (v_bytes) bulk_g2s(dst + q_bytes + k_bytes, static_cast<const T*>(a.v) + t * a.v_stride_t, v_bytes, &bars.full[s]);
    if (known && r_bytes) bulk_g2s(dst + q_bytes + k_bytes + v_bytes, a.table + int64_t(pos) * R, r_bytes, &bars.full[s]);
  };
  if (threadIdx.x == 0) {
    mbar_init(&bars.full[0], 1);
    mbar_init(&bars.full[1], 1);
    bars.dead = 0;
    fence_mbar_init();
  }
  __syncthreads();
  if (threadIdx.x < 32) {
    bring(blockIdx.x, 0);
    if (int64_t(blockIdx.x) + gridDim.x < batches) bring(int64_t(blockIdx.x) + gridDim.x, 1);
  }
  int turn = 0;
  int64_t n = blockIdx.x;
  for (; n < batches; n += gridDim.x, ++turn) {
    const int s = turn & 1, tokens = int(min(int64_t(p.per), a.n_tokens - n * p.per));
    const bool here = __all_sync(~0u, mbar_wait(&bars.full[s], (turn >> 1) & 1, p.spin));
    if (!here) bars.dead = 1;
    const uint8_t* base = smem + s * batch;
    if (here && v_bytes && int(threadIdx.x) < tokens) {  // values: straight on
      const int64_t t = n * p.per + threadIdx.x, at = slot_offset(p, a.slots[t]);
      if (at >= 0) {
        const uint32_t src = smem_u32(base) + threadIdx.x * token + q_bytes + k_bytes;
        if (a.c_stride_h == D) bulk_s2g(static_cast<T*>(a.v_cache) + at, src, v_bytes);
        else
          for (int h = 0; h < a.n_kv_heads; ++h) bulk_s2g(static_cast<T*>(a.v_cache) + at + h * a.c_stride_h, src + h * row, row);
      }
      asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    }
    if (here && mine < tokens) {
      const int64_t t = n * p.per + mine;
      const uint8_t* rows = base + mine * token;
      uint64_t c[4], sn[4];
      if (turned) {
        const float* cs = reinterpret_cast<const float*>(rows + q_bytes + k_bytes + v_bytes);
        if (bars.pos[s][mine] >= 0) {
          const float4* c4 = reinterpret_cast<const float4*>(cs + (INTERLEAVED ? ea / 2 : ea));
          const float4* d4 = reinterpret_cast<const float4*>(cs + (INTERLEAVED ? (ea + ahead) / 2 : ea + 4));
          const float4 c0 = c4[0], c1 = d4[0], s0 = c4[R / 8], s1 = d4[R / 8];
          c[0] = pair(c0.x, c0.y); c[1] = pair(c0.z, c0.w); c[2] = pair(c1.x, c1.y); c[3] = pair(c1.z, c1.w);
          sn[0] = pair(s0.x, s0.y); sn[1] = pair(s0.z, s0.w); sn[2] = pair(s1.x, s1.y); sn[3] = pair(s1.z, s1.w);
        } else {
          const float nan = __int_as_float(0x7FC00000);
#pragma unroll
          for (int e = 0; e < 4; ++e) c[e] = sn[e] = pair(nan, nan);
        }
      }
      auto turn_row = [&](const T* src, bool weighted, const uint64_t (&w)[8], T* dst, T* also) {
        uint64_t x[8] = {};
        if (live) {
          const Vec8<DT> va = load8s<DT>(src), vb = load8s<DT>(src + ahead);
          unpack8<DT>(va, x);
          unpack8<DT>(vb, x + 4);
        }
        if (weighted) {
          uint64_t sq[2] = {0, 0};
#pragma unroll
          for (int e = 0; e < 8; ++e) sq[e & 1] = fma2(x[e], x[e], sq[e & 1]);
          const float2 f = split(add2(sq[0], sq[1]));
          float ss = f.x + f.y;
#pragma unroll
          for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(mask, ss, o);
          const float r = rsqrtf(fmaf(ss, p.inv_dim, a.eps));
          const uint64_t r2 = pair(r, r);
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = mul2(x[e], mul2(r2, w[e]));
        }
        if (turned) rotate<INTERLEAVED>(x, c, sn);
        if (!live) return;
        const Vec8<DT> va = pack8<DT>(x), vb = pack8<DT>(x + 4);
        if (dst) {
          store8<DT>(dst, va);
          store8<DT>(dst + ahead, vb);
        }
        if (also) {
          store8<DT>(also, va);
          store8<DT>(also + ahead, vb);
        }
      };
      const T* q = reinterpret_cast<const T*>(rows) + ea;
      T* qo = static_cast<T*>(a.q_out) + t * a.n_q_heads * D + ea;
      int h = first;
      for (; h < a.n_q_heads; h += share) turn_row(q + h * D, a.q_weight != nullptr, wq, qo + h * D, nullptr);
      const int64_t at = a.k_cache ? slot_offset(p, a.slots[t]) : -1;
      T* kc = at < 0 ? nullptr : static_cast<T*>(a.k_cache) + at + ea;
      T* ko = a.k_out ? static_cast<T*>(a.k_out) + t * a.n_kv_heads * D + ea : nullptr;
      for (; h < a.n_q_heads + a.n_kv_heads; h += share) {  // keys follow the queries
        const int hk = h - a.n_q_heads;
        turn_row(q + h * D, a.k_weight != nullptr, wk, kc ? kc + hk * a.c_stride_h : nullptr, ko ? ko + hk * D : nullptr);
      }
    }
    // the stage is read (by the value copies too) before it is filled again
    if (v_bytes && int(threadIdx.x) < p.per) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
    fence_proxy_async_smem();
    __syncthreads();
    if (bars.dead) break;
    const int64_t next = n + 2 * int64_t(gridDim.x);
    if (threadIdx.x < 32 && next < batches) bring(next, s);
  }
  if (v_bytes && int(threadIdx.x) < p.per) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  if (!bars.dead) return;
  for (int i = 0; i < 2; ++i, n += gridDim.x, ++turn)  // this batch and the next are under way
    if (n < batches) mbar_drain(&bars.full[turn & 1], (turn >> 1) & 1);
  if (threadIdx.x == 0) atomicOr(&g_norm_rope_fault, 1u);
}

__global__ void __launch_bounds__(NR_THREADS) norm_rope_any_kernel(const __grid_constant__ NrParams p) {
  const smaq_norm_rope_args& a = p.a;
  const int lane = threadIdx.x & 31;
  const int64_t job = int64_t(blockIdx.x) * (NR_THREADS / 32) + (threadIdx.x >> 5);
  const int64_t t = job / p.heads;
  if (t >= a.n_tokens) return;
  const int h = int(job - t * p.heads), D = a.head_dim, R = a.rotary_dim, Hq = a.n_q_heads, Hk = a.n_kv_heads;
  const int kind = h < Hq ? 0 : h < Hq + Hk ? 1 : 2, hk = kind == 1 ? h - Hq : h - Hq - Hk;
  const void* src = kind == 0 ? a.q : kind == 1 ? a.k : a.v;
  const int64_t in = kind == 0   ? t * a.q_stride_t + h * a.q_stride_h
                     : kind == 1 ? t * a.k_stride_t + hk * a.k_stride_h
                                 : t * a.v_stride_t + hk * a.v_stride_h;
  const int64_t dst = a.k_cache ? slot_offset(p, a.slots[t]) : -1;
  auto put = [&](int e, float x) {
    if (kind == 0) store_elem(a.q_out, a.dtype, (t * Hq + h) * D + e, x);
    if (kind == 1 && a.k_out) store_elem(a.k_out, a.dtype, (t * Hk + hk) * D + e, x);
    if (kind > 0 && dst >= 0) store_elem(kind == 1 ? a.k_cache : a.v_cache, a.dtype, dst + hk * a.c_stride_h + e, x);
  };
  if (kind == 2) {
    for (int e = lane; e < D; e += 32) put(e, load_elem(src, a.dtype, in + e));
    return;
  }
  const float* weight = kind ? a.k_weight : a.q_weight;
  float r = 1.f;
  if (weight) {
    float ss = 0.f;
    for (int e = lane; e < D; e += 32) {
      const float x = load_elem(src, a.dtype, in + e);
      ss = fmaf(x, x, ss);
    }
    r = 1.0f / sqrtf(warp_sum(ss) / float(D) + a.eps);
  }
  auto normed = [&](int e) {
    const float x = load_elem(src, a.dtype, in + e);
    return weight ? x * (r * weight[e]) : x;
  };
  const int pos = a.positions[t];
  const bool known = pos >= 0 && pos < a.n_positions;
  for (int i = lane; i < R / 2; i += 32) {
    const int ea = a.interleaved ? 2 * i : i, eb = a.interleaved ? 2 * i + 1 : i + R / 2;
    const float c = known ? a.table[int64_t(pos) * R + i] : __int_as_float(0x7FC00000);
    const float s = known ? a.table[int64_t(pos) * R + R / 2 + i] : __int_as_float(0x7FC00000);
    const float u = normed(ea), v = normed(eb);
    put(ea, u * c - v * s);
    put(eb, v * c + u * s);
  }
  for (int e = R + lane; e < D; e += 32) put(e, normed(e));
}

// Tokens a batch of the staged kernel, 0 where it does not serve: heads side by side, batches of 32 KB or more, and tokens
// enough for three rounds of batches on every CTA.  Against the other kernel, with the cache write: 32/8 heads of 128,
// 16384 tokens 88 us / 101, 8192 (7 rounds) 49 / 54, 2000 (1.7) 16.5 / 15.8; 32/8 of 256, 4000 tokens 47 / 53; 12/4 of
// 64, 16000 tokens 30 / 33; 8/1 of 64, 16000 tokens in batches of 25 KB 26 / 21.  Near the crossover, at 3.5 rounds, 4096
// normed tokens of 32/8 heads of 128 with the cache write take 31 / 30, 4099 half-rotated ones without norm and cache 20.3 / 22.5.
int staged_tokens(const smaq_norm_rope_args& a, int size, int groups) {
  const bool cache = a.k_cache != nullptr;
  if (a.q_stride_h != a.head_dim || a.k_stride_h != a.head_dim || (cache && a.v_stride_h != a.head_dim)) return 0;
  const int64_t token = int64_t(a.n_q_heads + a.n_kv_heads * (cache ? 2 : 1)) * a.head_dim * size + a.rotary_dim * 4;
  const int64_t per = NS_SMEM / 2 / token;
  int two = 0;
  for (int i = 1; i <= per && i <= NS_MOST && i <= groups; i *= 2) two = i;  // the lane groups divide over the tokens
  return two * token >= 32 * 1024 && a.n_tokens >= int64_t(num_sms()) * NS_CTAS * NS_ROUNDS * two ? two : 0;
}

template <class DT, int LANES>
int launch_lanes(NrParams& p, cudaStream_t st) {
  if (const int per = staged_tokens(p.a, int(sizeof(typename DT::T)), NS_THREADS / LANES)) {
    p.per = per;
    const int64_t token = int64_t(p.heads) * p.a.head_dim * sizeof(typename DT::T) + p.a.rotary_dim * 4, batches = (p.a.n_tokens + per - 1) / per;
    auto kern = p.a.interleaved ? norm_rope_staged_kernel<DT, LANES, true> : norm_rope_staged_kernel<DT, LANES, false>;
    if (const int rc = allow_smem(reinterpret_cast<const void*>(kern), NS_SMEM, "norm_rope")) return rc;
    const int64_t most = int64_t(num_sms()) * NS_CTAS, grid = batches < most ? batches : most;
    kern<<<unsigned(grid), NS_THREADS, size_t(2 * token * per), st>>>(p);
    return cuda_status(cudaGetLastError(), "norm_rope");
  }
  const int64_t jobs = p.a.n_tokens * p.groups, per_cta = NR_THREADS / LANES, grid = (jobs + per_cta - 1) / per_cta;
  if (grid >= (int64_t(1) << 31)) return fail(SMAQ_ERR_UNSUPPORTED, "norm_rope: too many rows");
  if (p.a.interleaved) norm_rope_kernel<DT, LANES, true><<<unsigned(grid), NR_THREADS, 0, st>>>(p);
  else norm_rope_kernel<DT, LANES, false><<<unsigned(grid), NR_THREADS, 0, st>>>(p);
  return cuda_status(cudaGetLastError(), "norm_rope");
}
template <class DT>
int launch_dtype(NrParams& p, cudaStream_t st) {
  const int need = p.a.head_dim / 16;
  const int lanes = need <= 4 ? 4 : need <= 8 ? 8 : need <= 16 ? 16 : 32;
  // heads a lane group walks: all of them would read a token's cosines once, but few tokens must
  // spread over the GPU; aim at four CTAs of threads an SM
  const int64_t want = int64_t(num_sms()) * 4 * NR_THREADS / lanes;  // lane groups
  int64_t per = p.a.n_tokens * p.heads / want;
  p.per = int(per < 1 ? 1 : per > NR_PER ? NR_PER : per);
  p.q_groups = (p.a.n_q_heads + p.per - 1) / p.per;
  p.k_groups = (p.a.n_kv_heads + p.per - 1) / p.per;
  p.groups = p.q_groups + p.k_groups * (p.a.k_cache ? 2 : 1);
  switch (lanes) {
    case 4: return launch_lanes<DT, 4>(p, st);
    case 8: return launch_lanes<DT, 8>(p, st);
    case 16: return launch_lanes<DT, 16>(p, st);
    default: return launch_lanes<DT, 32>(p, st);
  }
}

}  // namespace

}  // namespace smaq

extern "C" int smaq_norm_rope(const smaq_norm_rope_args* args, void* stream) {
  using namespace smaq;
  if (!args) return fail(SMAQ_ERR_INVALID, "norm_rope: null arguments");
  const smaq_norm_rope_args& a = *args;
  if (a.dtype != SMAQ_F32 && a.dtype != SMAQ_BF16 && a.dtype != SMAQ_F16) return fail(SMAQ_ERR_INVALID, "norm_rope: dtype %d", a.dtype);
  if (a.n_tokens < 0 || a.n_q_heads < 1 || a.n_kv_heads < 1 || a.head_dim < 1)
    return fail(SMAQ_ERR_INVALID, "norm_rope: bad sizes (tokens %lld, heads %d/%d, head_dim %d)", (long long)a.n_tokens, a.n_q_heads,
                a.n_kv_heads, a.head_dim);
  if (a.rotary_dim < 0 || a.rotary_dim > a.head_dim || a.rotary_dim % 2)
    return fail(SMAQ_ERR_INVALID, "norm_rope: rotary_dim %d must be even and within head_dim %d", a.rotary_dim, a.head_dim);
  if (a.n_tokens == 0) return SMAQ_OK;
  if (!a.q || !a.k || !a.q_out || !a.positions || (a.rotary_dim && !a.table)) return fail(SMAQ_ERR_INVALID, "norm_rope: null pointer");
  const bool cache = a.k_cache || a.v_cache || a.v || a.slots;
  if (cache && (!a.k_cache || !a.v_cache || !a.v || !a.slots || a.page_size < 1 || a.n_pages < 0))
    return fail(SMAQ_ERR_INVALID, "norm_rope: a cache write needs v, both caches, slots and a page_size");
  if (!cache && !a.k_out) return fail(SMAQ_ERR_INVALID, "norm_rope: neither a cache nor k_out");
  NrParams p;
  p.a = a;
  p.heads = a.n_q_heads + a.n_kv_heads * (cache ? 2 : 1);
  p.spin = exact_wait_limit();
  p.per = 1;
  p.groups = p.heads;
  p.inv_dim = 1.0f / float(a.head_dim);
  p.page_div = make_fastdiv(cache ? a.page_size : 1);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t e = a.dtype == SMAQ_F32 ? 4 : 2;  // every vector on a 16-byte boundary
  auto aligned = [&](const void* ptr, int64_t s1, int64_t s2, int64_t s3) {
    return reinterpret_cast<uintptr_t>(ptr) % 16 == 0 && (s1 * e) % 16 == 0 && (s2 * e) % 16 == 0 && (s3 * e) % 16 == 0;
  };
  const bool fast = a.head_dim % 16 == 0 && a.head_dim <= 512 && a.rotary_dim % 16 == 0 &&
                    aligned(a.q, a.q_stride_t, a.q_stride_h, 0) && aligned(a.k, a.k_stride_t, a.k_stride_h, 0) &&
                    aligned(a.q_out, 0, 0, 0) && aligned(a.k_out, 0, 0, 0) && reinterpret_cast<uintptr_t>(a.table) % 16 == 0 &&
                    reinterpret_cast<uintptr_t>(a.q_weight) % 16 == 0 && reinterpret_cast<uintptr_t>(a.k_weight) % 16 == 0 &&
                    (!cache || (aligned(a.v, a.v_stride_t, a.v_stride_h, 0) &&
                                aligned(a.k_cache, a.c_stride_page, a.c_stride_slot, a.c_stride_h) && aligned(a.v_cache, 0, 0, 0)));
  if (!fast) {
    const int64_t jobs = a.n_tokens * p.heads, grid = (jobs + NR_THREADS / 32 - 1) / (NR_THREADS / 32);
    if (grid >= (int64_t(1) << 31)) return fail(SMAQ_ERR_UNSUPPORTED, "norm_rope: too many rows");
    norm_rope_any_kernel<<<unsigned(grid), NR_THREADS, 0, st>>>(p);
    return cuda_status(cudaGetLastError(), "norm_rope");
  }
  switch (a.dtype) {
    case SMAQ_F32: return launch_dtype<F32>(p, st);
    case SMAQ_BF16: return launch_dtype<BF16>(p, st);
    default: return launch_dtype<F16>(p, st);
  }
}

namespace smaq {
int norm_rope_fault(bool& set) {
  unsigned int word = 0, zero = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&word, g_norm_rope_fault, sizeof(word));
  if (e == cudaSuccess && word) e = cudaMemcpyToSymbol(g_norm_rope_fault, &zero, sizeof(zero));
  set = word != 0;
  return cuda_status(e, "exact status: read");
}
}  // namespace smaq
