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
// when there are enough tokens to fill the GPU, and loads two heads ahead.  Values are copied by the same
// walk.  Bound by HBM bytes for prompts, by latency for decode steps.
// norm_rope_any_kernel: any head_dim and alignment, one warp a head, element by element.
#include "common.cuh"

namespace smaq {

namespace {

struct NrParams {
  smaq_norm_rope_args a;
  int heads;            // q + k (+ v with a cache)
  int per;              // heads that a lane group walks
  int groups;           // ceil(heads / per)
  FastDiv page_div;
};

constexpr int NR_THREADS = 256;

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
__device__ __forceinline__ void store8(typename DT::T* p, const Vec8<DT>& v) {
  *reinterpret_cast<decltype(v.u)*>(p) = v.u;
  if constexpr (DT::code == SMAQ_F32) reinterpret_cast<float4*>(p)[1] = v.w;
}
template <class DT>
__device__ __forceinline__ void unpack8(const Vec8<DT>& v, float* x) {
  const typename DT::T* e = reinterpret_cast<const typename DT::T*>(&v);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = to_f(e[i]);
}
template <class DT>
__device__ __forceinline__ Vec8<DT> pack8(const float* x) {
  Vec8<DT> v;
  typename DT::T* e = reinterpret_cast<typename DT::T*>(&v);
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i] = from_f<DT>(x[i]);
  return v;
}
__device__ __forceinline__ void load8f(const float* p, float* x) {
  const float4 u = __ldg(reinterpret_cast<const float4*>(p)), w = __ldg(reinterpret_cast<const float4*>(p) + 1);
  x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w;
  x[4] = w.x; x[5] = w.y; x[6] = w.z; x[7] = w.w;
}

// LANES lanes a head (a power of two >= head_dim / 16).
template <class DT, int LANES, bool INTERLEAVED>
__global__ void __launch_bounds__(NR_THREADS) norm_rope_kernel(const __grid_constant__ NrParams p) {
  using T = typename DT::T;
  const smaq_norm_rope_args& a = p.a;
  const int lane = threadIdx.x % LANES;
  const int64_t job = int64_t(blockIdx.x) * (NR_THREADS / LANES) + threadIdx.x / LANES;
  const int64_t t = job / p.groups;
  if (t >= a.n_tokens) return;  // whole lane groups leave; the shuffles below name the group's lanes
  const unsigned mask = (LANES == 32 ? ~0u : ((1u << LANES) - 1u) << ((threadIdx.x & 31) / LANES * LANES));
  const int h0 = int(job - t * p.groups) * p.per, h1 = min(h0 + p.per, p.heads);
  const int D = a.head_dim, R = a.rotary_dim, Hq = a.n_q_heads, Hk = a.n_kv_heads;
  const bool live = lane < D / 16, turned = lane < R / 16;
  // this lane's two vectors
  const int ea = turned ? 8 * lane : R + 16 * (lane - R / 16), eb = turned ? R / 2 + 8 * lane : ea + 8;

  float c[16], s[16];
  if (turned && h0 < Hq + Hk) {
    const int pos = a.positions[t];
    if (pos >= 0 && pos < a.n_positions) {
      const float* row = a.table + int64_t(pos) * R;
      if constexpr (INTERLEAVED) {
        // pair i of vector a (b) is pair ea / 2 + i (eb / 2 + i)
        const float4 ca = __ldg(reinterpret_cast<const float4*>(row + ea / 2)), cb = __ldg(reinterpret_cast<const float4*>(row + eb / 2));
        const float4 sa = __ldg(reinterpret_cast<const float4*>(row + R / 2 + ea / 2)), sb = __ldg(reinterpret_cast<const float4*>(row + R / 2 + eb / 2));
        c[0] = ca.x; c[1] = ca.y; c[2] = ca.z; c[3] = ca.w; c[4] = cb.x; c[5] = cb.y; c[6] = cb.z; c[7] = cb.w;
        s[0] = sa.x; s[1] = sa.y; s[2] = sa.z; s[3] = sa.w; s[4] = sb.x; s[5] = sb.y; s[6] = sb.z; s[7] = sb.w;
      } else {
        load8f(row + ea, c);
        load8f(row + R / 2 + ea, s);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) c[i] = s[i] = __int_as_float(0x7FC00000);
    }
  }
  const int64_t dst = a.k_cache ? slot_offset(p, a.slots[t]) : 0;
  float w[16];
  int weighted = -1;  // whose weights w holds: 0 queries, 1 keys

  auto source = [&](int h) {
    return h < Hq        ? static_cast<const T*>(a.q) + t * a.q_stride_t + h * a.q_stride_h
           : h < Hq + Hk ? static_cast<const T*>(a.k) + t * a.k_stride_t + (h - Hq) * a.k_stride_h
                         : static_cast<const T*>(a.v) + t * a.v_stride_t + (h - Hq - Hk) * a.v_stride_h;
  };
  auto finish = [&](int h, Vec8<DT> va, Vec8<DT> vb) {
    if (h < Hq + Hk) {
      const int kind = h >= Hq;
      const float* weight = kind ? a.k_weight : a.q_weight;
      float x[16];
      unpack8(va, x);
      unpack8(vb, x + 8);
      if (weight) {
        if (weighted != kind) {
          weighted = kind;
          if (live) {
            load8f(weight + ea, w);
            load8f(weight + eb, w + 8);
          }
        }
        float ss = 0.f;
        if (live) {
#pragma unroll
          for (int i = 0; i < 16; ++i) ss = fmaf(x[i], x[i], ss);
        }
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(mask, ss, o);
        const float r = 1.0f / sqrtf(ss / float(D) + a.eps);
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] *= r * w[i];
      }
      if (turned) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          // pair i: (i, i + 8) of this lane's sixteen, or its neighbours (2i, 2i + 1)
          const int ia = INTERLEAVED ? 2 * i : i, ib = INTERLEAVED ? 2 * i + 1 : i + 8;
          const float u = x[ia], v = x[ib];
          x[ia] = u * c[i] - v * s[i];
          x[ib] = v * c[i] + u * s[i];
        }
      }
      va = pack8<DT>(x);
      vb = pack8<DT>(x + 8);
    }
    if (!live) return;
    if (h < Hq) {
      T* o = static_cast<T*>(a.q_out) + (t * Hq + h) * D;
      store8<DT>(o + ea, va);
      store8<DT>(o + eb, vb);
      return;
    }
    const int hk = h < Hq + Hk ? h - Hq : h - Hq - Hk;
    if (h < Hq + Hk && a.k_out) {
      T* o = static_cast<T*>(a.k_out) + (t * Hk + hk) * D;
      store8<DT>(o + ea, va);
      store8<DT>(o + eb, vb);
    }
    if (a.k_cache && dst >= 0) {
      T* o = static_cast<T*>(h < Hq + Hk ? a.k_cache : a.v_cache) + dst + hk * a.c_stride_h;
      store8<DT>(o + ea, va);
      store8<DT>(o + eb, vb);
    }
  };

  Vec8<DT> zero = {};
  for (int h = h0; h < h1; h += 2) {
    const bool two = h + 1 < h1;
    Vec8<DT> a0 = zero, b0 = zero, a1 = zero, b1 = zero;
    if (live) {
      const T* s0 = source(h);
      a0 = load8<DT>(s0 + ea);
      b0 = load8<DT>(s0 + eb);
      if (two) {
        const T* s1 = source(h + 1);
        a1 = load8<DT>(s1 + ea);
        b1 = load8<DT>(s1 + eb);
      }
    }
    finish(h, a0, b0);
    if (two) finish(h + 1, a1, b1);
  }
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

template <class DT, int LANES>
int launch_lanes(const NrParams& p, cudaStream_t st) {
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
  per = per < 1 ? 1 : per > 8 ? 8 : per;
  p.groups = int((p.heads + per - 1) / per);
  p.per = (p.heads + p.groups - 1) / p.groups;
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
  p.per = 1;
  p.groups = p.heads;
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
