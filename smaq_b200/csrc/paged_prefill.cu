// Attention of prompt chunks over the exact paged cache: causal behind any cached context, with a window,
// a prefix that all rows see, capped scores and a distance bias.
//
// A CTA takes one tile of rows of one request and KV head (rows = tokens times the query heads of the group, so
// grouped heads share every key and value that is brought on chip) and walks the tokens that some row of it
// sees, with a running maximum and sum per row.  The tiles of all requests are numbered from cu_query on the
// GPU; the host knows only the number of rows.  Tiles with the longest walks start first.
//
// prefill_tc.cu (bf16 / fp16, head_dim 64 / 128 / 256): the tensor-core kernel, everything but tables of one block.
// prefill_mma_kernel (the same types and head dims, tables of up to 128 tokens): four warps of 16 rows, m16n8k16 products, blocks of
//   64 (head_dim 256: 32) tokens brought by cp.async into two stages, page lookups two blocks ahead.
// prefill_fma_kernel, prefill_simt_kernel (fp32, other head dims and alignments): tiles of 64 rows by 64 tokens, or,
//   with few rows, of four rows and 16 lane groups with a token each; all arithmetic in 32 bits.
#include "paged_prefill.cuh"
#include "prefill_tc.cuh"

namespace smaq {

namespace {

constexpr int PM_THREADS = 128;

template <int D>
struct PmCfg {
  static constexpr int ROWS = 64;
  static constexpr int N = D == 256 ? 32 : 64;       // tokens a block
  static constexpr int Q = ROWS * D * 2;
  static constexpr int STAGE = 2 * N * D * 2;
  static constexpr int SMEM = Q + 2 * STAGE;
};

template <class DT, int D, int CAP>
__global__ void __launch_bounds__(PM_THREADS, 2) prefill_mma_kernel(const __grid_constant__ PagedParams p) {
  using T = typename DT::T;
  constexpr int N = PmCfg<D>::N, STAGE = PmCfg<D>::STAGE, CH = D / 8, NT = D / 8;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int64_t offs[2][N];
  __shared__ int sums[PM_THREADS / 32];
  __shared__ PrefillTile found;
  const smaq_paged_args& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, kvh = blockIdx.y;
  write_padding(p, kvh, blockIdx.x, gridDim.x);
  const PrefillTile t = find_tile<PM_THREADS>(p, blockIdx.x, PmCfg<D>::ROWS, true, sums, &found);
  if (t.rows == 0) return;
  const PrefillBlocks blocks(t, N);
  const uint32_t qs = smem_u32(smem), ring = qs + PmCfg<D>::Q;
  const int32_t* table = a.block_table + t.b * a.table_stride;

  for (int i = threadIdx.x; i < PmCfg<D>::ROWS * CH; i += PM_THREADS) {
    const int r = i / CH, ch = i % CH, f = t.f0 + r, tok = fast_div(f, p.group_div);
    const bool live = r < t.rows;
    const T* src = static_cast<const T*>(a.q) + (live ? (t.first + tok) * a.q_stride_t + (kvh * p.group + f - tok * p.group) * a.q_stride_h + ch * 8 : 0);
    cp_async16(qs + uint32_t(r * D * 2 + ((ch ^ (r & 7)) << 4)), src, live ? 16u : 0u);
  }
  auto look_up = [&](int k) {
    if (k >= blocks.count || threadIdx.x >= N) return;
    const int j = blocks.base(k, N) + threadIdx.x;
    offs[k & 1][threadIdx.x] = tile_sees(t, j) ? token_offset(p, table, j) + kvh * a.c_stride_h : -1;
  };
  auto issue = [&](int k) {
    if (k < blocks.count) {
      const uint32_t st = ring + (k & 1) * STAGE;
#pragma unroll
      for (int i = 0; i < N * CH / PM_THREADS; ++i) {
        const int r = (i * PM_THREADS + threadIdx.x) / CH, ch = (i * PM_THREADS + threadIdx.x) % CH;
        const int64_t off = offs[k & 1][r], from = (off < 0 ? 0 : off) + ch * 8;
        const uint32_t at = st + uint32_t(r * D * 2 + ((ch ^ (r & 7)) << 4)), n = off < 0 ? 0u : 16u;
        cp_async16(at, static_cast<const T*>(a.k_cache) + from, n);
        cp_async16(at + N * D * 2, static_cast<const T*>(a.v_cache) + from, n);
      }
    }
    cp_async_commit();
  };

  // this thread's two rows
  const int f0 = t.f0 + warp * 16 + (lane >> 2), f1 = f0 + 8;
  const int t0 = fast_div(f0, p.group_div), t1 = fast_div(f1, p.group_div);
  const int i0 = t.past + t0, i1 = t.past + t1;
  const int h0 = kvh * p.group + f0 - t0 * p.group, h1 = kvh * p.group + f1 - t1 * p.group;
  const int last = t.f0 + t.rows;
  const float s0 = a.slopes && f0 < last ? a.slopes[h0] * kLog2e : 0.f, s1 = a.slopes && f1 < last ? a.slopes[h1] * kLog2e : 0.f;
  const int least = t.past + fast_div(t.f0, p.group_div), most = t.past + fast_div(last - 1, p.group_div);
  float o[NT][4] = {}, m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
  bool special = false;  // an infinite or NaN value in a block that is not seen by all rows

  look_up(0);
  __syncthreads();
  issue(0);
  look_up(1);
#pragma unroll 1
  for (int k = 0; k < blocks.count; ++k) {
    __syncthreads();  // the lookups of block k + 1 are there, its stage is free
    issue(k + 1);
    look_up(k + 2);
    cp_async_wait<1>();
    __syncthreads();
    const uint32_t ks = ring + (k & 1) * STAGE, vs = ks + N * D * 2;
    const int base = blocks.base(k, N);
    float c[N / 8][4] = {};
    const int qr = warp * 16 + (lane & 15), qc = lane >> 4;
    const int kr = (lane & 7) + ((lane >> 4) << 3), kc = (lane >> 3) & 1;
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
      uint32_t q[4];
      ldmatrix4(q, qs + uint32_t(qr * D * 2 + (((2 * s + qc) ^ (qr & 7)) << 4)));
#pragma unroll
      for (int n = 0; n < N / 16; ++n) {
        uint32_t b[4];
        ldmatrix4(b, ks + uint32_t((n * 16 + kr) * D * 2 + (((2 * s + kc) ^ (kr & 7)) << 4)));
        mma_16816<DT>(c[2 * n], q, b[0], b[1]);
        mma_16816<DT>(c[2 * n + 1], q, b[2], b[3]);
      }
    }
    const bool all = base + N <= t.prefix || (base + N <= least + 1 && (a.window == 0 || base > most - a.window));
    if (!all) {
      for (int i = threadIdx.x; i < N * CH; i += PM_THREADS) special |= any_special<DT>(*reinterpret_cast<const uint4*>(smem + (vs - qs) + i * 16));
    }
    float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
    for (int n = 0; n < N / 8; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int j = base + n * 8 + 2 * (lane & 3) + e;
        float x0 = score_log2<CAP>(c[n][e], p), x1 = score_log2<CAP>(c[n][2 + e], p);
        if (a.slopes) {
          x0 -= s0 * fabsf(float(i0 - j));
          x1 -= s1 * fabsf(float(i1 - j));
        }
        if (!all) {
          x0 = j < t.len && row_sees(p, t, i0, j) ? x0 : -INFINITY;
          x1 = j < t.len && row_sees(p, t, i1, j) ? x1 : -INFINITY;
        }
        c[n][e] = x0;
        c[n][2 + e] = x1;
        mx0 = fmaxf(mx0, x0);
        mx1 = fmaxf(mx1, x1);
      }
#pragma unroll
    for (int w = 1; w < 4; w <<= 1) {
      mx0 = fmaxf(mx0, __shfl_xor_sync(~0u, mx0, w));
      mx1 = fmaxf(mx1, __shfl_xor_sync(~0u, mx1, w));
    }
    mx0 -= kUp<DT>;
    mx1 -= kUp<DT>;
    if (__any_sync(~0u, mx0 > m0 || mx1 > m1)) {
      const float n0 = fmaxf(m0, mx0), n1 = fmaxf(m1, mx1);
      const float g0 = m0 == -INFINITY ? 0.f : ex2(m0 - n0), g1 = m1 == -INFINITY ? 0.f : ex2(m1 - n1);
      m0 = n0;
      m1 = n1;
      l0 *= g0;
      l1 *= g1;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        o[n][0] *= g0;
        o[n][1] *= g0;
        o[n][2] *= g1;
        o[n][3] *= g1;
      }
    }
    const float z0 = m0 == -INFINITY ? 0.f : m0, z1 = m1 == -INFINITY ? 0.f : m1;
    const int vr = (lane & 7) + (((lane >> 3) & 1) << 3), vc = lane >> 4;
#pragma unroll
    for (int s = 0; s < N / 16; ++s) {
      uint32_t w[4];
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const float* x = c[2 * s + n];
        const float p00 = ex2(x[0] - z0), p01 = ex2(x[1] - z0), p10 = ex2(x[2] - z1), p11 = ex2(x[3] - z1);
        l0 += p00 + p01;
        l1 += p10 + p11;
        w[2 * n] = pack2<DT>(p00, p01);
        w[2 * n + 1] = pack2<DT>(p10, p11);
      }
#pragma unroll
      for (int n = 0; n < NT / 2; ++n) {
        uint32_t b[4];
        ldmatrix4_trans(b, vs + uint32_t((s * 16 + vr) * D * 2 + (((2 * n + vc) ^ (vr & 7)) << 4)));
        mma_16816<DT>(o[2 * n], w, b[0], b[1]);
        mma_16816<DT>(o[2 * n + 1], w, b[2], b[3]);
      }
    }
  }
  cp_async_wait<0>();
  l0 += __shfl_xor_sync(~0u, l0, 1);
  l1 += __shfl_xor_sync(~0u, l1, 1);
  l0 += __shfl_xor_sync(~0u, l0, 2);
  l1 += __shfl_xor_sync(~0u, l1, 2);
  const float v0 = l0 == 0.f ? 0.f : 1.0f / l0, v1 = l1 == 0.f ? 0.f : 1.0f / l1;
  T* out = static_cast<T*>(a.out) + 2 * (lane & 3);
  T* o0 = out + (t.first + t0) * a.o_stride_t + h0 * a.o_stride_h;
  T* o1 = out + (t.first + t1) * a.o_stride_t + h1 * a.o_stride_h;
  float fine0 = 0.f, fine1 = 0.f;  // zero, or NaN where an output is not finite
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const float x0 = o[n][0] * v0, x1 = o[n][1] * v0, y0 = o[n][2] * v1, y1 = o[n][3] * v1;
    if (f0 < last) *reinterpret_cast<uint32_t*>(o0 + n * 8) = pack2<DT>(x0, x1);
    if (f1 < last) *reinterpret_cast<uint32_t*>(o1 + n * 8) = pack2<DT>(y0, y1);
    fine0 += (x0 + x1) * 0.f;
    fine1 += (y0 + y1) * 0.f;
  }
  if (a.lse && (lane & 3) == 0) {
    if (f0 < last) a.lse[int64_t(t.first + t0) * a.n_q_heads + h0] = (m0 + log2f(l0)) * kLn2;
    if (f1 < last) a.lse[int64_t(t.first + t1) * a.n_q_heads + h1] = (m1 + log2f(l1)) * kLn2;
  }
  if (__syncthreads_or(special)) {
    const uint32_t redo0 = __ballot_sync(~0u, fine0 != 0.f && l0 == l0), redo1 = __ballot_sync(~0u, fine1 != 0.f && l1 == l1);
    for (int r = 0; r < 16; ++r) {
      const int f = t.f0 + warp * 16 + r;
      if (((r < 8 ? redo0 : redo1) >> (4 * (r & 7)) & 15u) && f < last) exact_row(p, t, kvh, f);
    }
  }
}

// ---------------------------------------------------------------- other types, head dims and alignments
constexpr int PX_ROWS = 4;

template <class DT, int NI, bool VEC>
__global__ void __launch_bounds__(PM_THREADS) prefill_simt_kernel(const __grid_constant__ PagedParams p) {
  using T = typename DT::T;
  constexpr int GROUPS = PM_THREADS / 8, WARPS = PM_THREADS / 32;
  __shared__ __align__(16) float qs[PX_ROWS][32 * NI];
  __shared__ float acc[WARPS][PX_ROWS][32 * NI + 2];
  __shared__ int sums[WARPS];
  __shared__ PrefillTile found;
  const smaq_paged_args& a = p.a;
  const int D = a.head_dim, l = threadIdx.x & 7, grp = threadIdx.x >> 3, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, kvh = blockIdx.y;
  write_padding(p, kvh, blockIdx.x, gridDim.x);
  const PrefillTile t = find_tile<PM_THREADS>(p, blockIdx.x, PX_ROWS, true, sums, &found);
  if (t.rows == 0) return;
  for (int i = threadIdx.x; i < PX_ROWS * 32 * NI; i += PM_THREADS) {
    const int r = i / (32 * NI), e = i % (32 * NI), f = t.f0 + r, tok = f / p.group;
    qs[r][e] = r < t.rows && e < D ? load_elem(a.q, a.dtype, (t.first + tok) * a.q_stride_t + (kvh * p.group + f % p.group) * a.q_stride_h + e) : 0.f;
  }
  __syncthreads();
  float o[PX_ROWS][NI][4] = {}, m[PX_ROWS], s[PX_ROWS], slope[PX_ROWS];
  int pos[PX_ROWS];
#pragma unroll
  for (int r = 0; r < PX_ROWS; ++r) {
    const int f = t.f0 + r;
    m[r] = -INFINITY;
    s[r] = 0.f;
    pos[r] = r < t.rows ? t.past + f / p.group : -1;
    slope[r] = a.slopes && r < t.rows ? a.slopes[kvh * p.group + f % p.group] : 0.f;
  }
  const PrefillBlocks blocks(t, GROUPS);
  const int32_t* table = a.block_table + t.b * a.table_stride;
  const T* kc = static_cast<const T*>(a.k_cache) + kvh * a.c_stride_h;
  const T* vc = static_cast<const T*>(a.v_cache) + kvh * a.c_stride_h;
  for (int b = 0; b < blocks.count; ++b) {
    const int j = blocks.base(b, GROUPS) + grp;
    const bool seen = tile_sees(t, j);
    float k[NI][4], v[NI][4];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int e = 4 * (l + 8 * i);
#pragma unroll
      for (int x = 0; x < 4; ++x) k[i][x] = v[i][x] = 0.f;
      if (!seen) continue;
      const int64_t off = token_offset(p, table, j);
      if constexpr (VEC) {
        if (e < D) {
          load_vec<DT, 4>(kc + off + e, k[i]);
          load_vec<DT, 4>(vc + off + e, v[i]);
        }
      } else {
#pragma unroll
        for (int x = 0; x < 4; ++x)
          if (e + x < D) {
            k[i][x] = to_f(kc[off + e + x]);
            v[i][x] = to_f(vc[off + e + x]);
          }
      }
    }
#pragma unroll
    for (int r = 0; r < PX_ROWS; ++r) {
      float x = 0.f;
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const float4 q = *reinterpret_cast<const float4*>(&qs[r][4 * (l + 8 * i)]);
        x = fmaf(q.x, k[i][0], fmaf(q.y, k[i][1], fmaf(q.z, k[i][2], fmaf(q.w, k[i][3], x))));
      }
#pragma unroll
      for (int w = 1; w < 8; w <<= 1) x += __shfl_xor_sync(~0u, x, w);
      x *= a.scale;
      if (a.softcap > 0.f) x = a.softcap * tanhf(x / a.softcap);
      x = (x - slope[r] * fabsf(float(pos[r] - j))) * kLog2e;
      if (!seen || !row_sees(p, t, pos[r], j)) continue;
      if (x > m[r]) {
        const float f = ex2(m[r] - x);
        m[r] = x;
        s[r] *= f;
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[r][i][e] *= f;
      }
      const float w = ex2(x - (m[r] == -INFINITY ? 0.f : m[r]));
      s[r] += w;
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[r][i][e] = fmaf(w, v[i][e], o[r][i][e]);
    }
  }
#pragma unroll
  for (int r = 0; r < PX_ROWS; ++r) {
#pragma unroll
    for (int w = 8; w < 32; w <<= 1) {
      const float om = __shfl_xor_sync(~0u, m[r], w), os = __shfl_xor_sync(~0u, s[r], w);
      const float nm = fmaxf(m[r], om), z = nm == -INFINITY ? 0.f : nm, f = ex2(m[r] - z), g = ex2(om - z);
      m[r] = nm;
      s[r] = s[r] * f + os * g;
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[r][i][e] = o[r][i][e] * f + __shfl_xor_sync(~0u, o[r][i][e], w) * g;
    }
    if (lane < 8) {
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[warp][r][4 * (l + 8 * i) + e] = o[r][i][e];
      if (l == 0) {
        acc[warp][r][32 * NI] = m[r];
        acc[warp][r][32 * NI + 1] = s[r];
      }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < t.rows * D; i += PM_THREADS) {
    const int r = i / D, e = i - r * D, f = t.f0 + r, tok = f / p.group, h = kvh * p.group + f % p.group;
    float mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) mm = fmaxf(mm, acc[w][r][32 * NI]);
    const float z = mm == -INFINITY ? 0.f : mm;
    float x = 0.f, sum = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float g = ex2(acc[w][r][32 * NI] - z);
      x += g * acc[w][r][e];
      sum += g * acc[w][r][32 * NI + 1];
    }
    store_elem(a.out, a.dtype, int64_t(t.first + tok) * a.o_stride_t + h * a.o_stride_h + e, sum == 0.f ? 0.f : x / sum);
    if (a.lse && e == 0) a.lse[int64_t(t.first + tok) * a.n_q_heads + h] = (mm + log2f(sum)) * kLn2;
  }
}

// ---------------------------------------------------------------- many rows in 32 bits
// Tiles of 64 rows by blocks of 64 tokens in shared memory as 32-bit values, both products by FMA: a thread has 4 x 4
// scores, then 4 rows by DP / 16 channels (DP: head_dim rounded up to 64).  2048 fp32 tokens at 32/8 heads of 128:
// 1279 us, 27 TFLOP/s (four-row tiles: 3950 us), bound by the reads of shared memory (two float4 for 16 FMAs a thread)
// and the loads between the products; eight rows a thread, with half the warps, take 1290 us.
// Every product, weight and sum is fp32: tensor-core products would round the operands.
constexpr int64_t NO_SLOT = INT64_MIN;  // a token that no row sees
constexpr int PF_THREADS = 256, PF_STEP = PF_THREADS / 16, PF_ROWS = 64, PF_N = 64, PF_LD = 68;  // PF_LD: 64 and a pad that keeps float4 aligned

template <int DP>
constexpr int pf_smem() { return (2 * DP * PF_LD + PF_N * DP + (DP > 128 ? PF_N * PF_LD : 0)) * 4; }

template <class DT, int DP, bool VEC>
__global__ void __launch_bounds__(PF_THREADS, DP <= 128 ? 2 : 1) prefill_fma_kernel(const __grid_constant__ PagedParams p) {
  using T = typename DT::T;
  constexpr int NI = DP / 64, U = 8;  // U: loads in flight a thread
  extern __shared__ __align__(16) float sm[];
  __shared__ int64_t offs[2][PF_N];
  float *qs = sm, *ks = qs + DP * PF_LD, *vs = ks + DP * PF_LD, *ps = DP > 128 ? vs + PF_N * DP : ks;  // up to 128 the weights take the keys' place: two CTAs an SM
  __shared__ int sums[PF_THREADS / 32];
  __shared__ PrefillTile found;
  const smaq_paged_args& a = p.a;
  const int D = a.head_dim, tid = threadIdx.x, tx = tid & 15, ty = tid >> 4, kvh = blockIdx.y;
  write_padding(p, kvh, blockIdx.x, gridDim.x);
  const PrefillTile t = find_tile<PF_THREADS>(p, blockIdx.x, PF_ROWS, true, sums, &found);
  if (t.rows == 0) return;
  const PrefillBlocks blocks(t, PF_N);
  const int32_t* table = a.block_table + t.b * a.table_stride;
  auto load4 = [&](const T* row, int e, float (&x)[4]) {  // elements e .. e + 3 of a row, zeros past its end
    if constexpr (VEC) {
      if (e < D) load_vec<DT, 4>(row + e, x);
      else x[0] = x[1] = x[2] = x[3] = 0.f;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = e + i < D ? to_f(row[e + i]) : 0.f;
    }
  };
  auto find_slots = [&](int b) {  // where a block's tokens lie
    if (tid < PF_N) {
      const int j = blocks.base(b, PF_N) + tid;
      offs[b & 1][tid] = tile_sees(t, j) ? token_offset(p, table, j) + kvh * a.c_stride_h : NO_SLOT;
    }
  };
  find_slots(0);
  const int last = t.f0 + t.rows, least = t.past + fast_div(t.f0, p.group_div), most = t.past + fast_div(last - 1, p.group_div);
  {
    const int r = tid & 63, f = t.f0 + r, tok = fast_div(f, p.group_div);
    const T* src = static_cast<const T*>(a.q) + (f < last ? int64_t(t.first + tok) * a.q_stride_t + (kvh * p.group + f - tok * p.group) * a.q_stride_h : 0);
    for (int e = (tid >> 6) * 4; e < DP; e += PF_STEP) {
      float x[4] = {};
      if (f < last) load4(src, e, x);
#pragma unroll
      for (int i = 0; i < 4; ++i) qs[(e + i) * PF_LD + r] = x[i];
    }
  }
  int pos[4], head[4];
  float slope[4], m[4], l[4], o[4][NI * 4];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int f = t.f0 + ty * 4 + r, tok = fast_div(f, p.group_div);
    pos[r] = t.past + tok;
    head[r] = kvh * p.group + f - tok * p.group;
    slope[r] = a.slopes && f < last ? a.slopes[head[r]] : 0.f;
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int c = 0; c < NI * 4; ++c) o[r][c] = 0.f;
  }
  bool special = false;
  for (int b = 0; b < blocks.count; ++b) {
    const int base = blocks.base(b, PF_N);
    const bool all = base + PF_N <= t.prefix || (base + PF_N <= least + 1 && (a.window == 0 || base > most - a.window));
    __syncthreads();  // the block before is read
    {  // keys: a token a lane, transposed
      const int r = tid & 63;
      const int64_t off = offs[b & 1][r];
#pragma unroll 1
      for (int e0 = (tid >> 6) * 4; e0 < DP; e0 += U * PF_STEP) {
        float x[U][4] = {};
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (off != NO_SLOT && e0 + u * PF_STEP < DP) load4(static_cast<const T*>(a.k_cache) + off, e0 + u * PF_STEP, x[u]);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (e0 + u * PF_STEP < DP) ks[(e0 + u * PF_STEP + i) * PF_LD + r] = x[u][i];
      }
    }
#pragma unroll 1
    for (int i0 = tid; i0 < PF_N * (DP / 4); i0 += U * PF_THREADS) {
      float x[U][4] = {};
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * PF_THREADS;
        const int64_t off = offs[b & 1][i / (DP / 4) % PF_N];
        if (off != NO_SLOT && i < PF_N * (DP / 4)) load4(static_cast<const T*>(a.v_cache) + off, i % (DP / 4) * 4, x[u]);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * PF_THREADS;
        if (!all) special |= !(fabsf(x[u][0]) + fabsf(x[u][1]) + fabsf(x[u][2]) + fabsf(x[u][3]) < INFINITY);
        if (i < PF_N * (DP / 4)) *reinterpret_cast<float4*>(vs + i / (DP / 4) * DP + i % (DP / 4) * 4) = make_float4(x[u][0], x[u][1], x[u][2], x[u][3]);
      }
    }
    __syncthreads();
    if (b + 1 < blocks.count) find_slots(b + 1);
    float s[4][4] = {};
#pragma unroll 8
    for (int e = 0; e < DP; ++e) {
      const float4 q = *reinterpret_cast<const float4*>(qs + e * PF_LD + ty * 4), k = *reinterpret_cast<const float4*>(ks + e * PF_LD + tx * 4);
      const float qv[4] = {q.x, q.y, q.z, q.w}, kv[4] = {k.x, k.y, k.z, k.w};
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < 4; ++c) s[r][c] = fmaf(qv[r], kv[c], s[r][c]);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      float mx = -INFINITY;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int j = base + tx * 4 + c;
        float x = s[r][c] * a.scale;
        if (a.softcap > 0.f) x = a.softcap * tanhf(x / a.softcap);
        if (a.slopes) x -= slope[r] * fabsf(float(pos[r] - j));
        x *= kLog2e;
        s[r][c] = all || (j < t.len && row_sees(p, t, pos[r], j)) ? x : -INFINITY;
        mx = fmaxf(mx, s[r][c]);
      }
#pragma unroll
      for (int w = 1; w < 16; w <<= 1) mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, w));
      if (mx > m[r]) {  // alike for the sixteen threads of a row
        const float f = ex2(m[r] - mx);
        m[r] = mx;
        l[r] *= f;
#pragma unroll
        for (int c = 0; c < NI * 4; ++c) o[r][c] *= f;
      }
      const float z = m[r] == -INFINITY ? 0.f : m[r];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        s[r][c] = ex2(s[r][c] - z);
        l[r] += s[r][c];
      }
    }
    if (DP <= 128) __syncthreads();  // the keys are read
#pragma unroll
    for (int c = 0; c < 4; ++c) *reinterpret_cast<float4*>(ps + (tx * 4 + c) * PF_LD + ty * 4) = make_float4(s[0][c], s[1][c], s[2][c], s[3][c]);
    __syncthreads();
#pragma unroll 4
    for (int j = 0; j < PF_N; ++j) {
      const float4 w = *reinterpret_cast<const float4*>(ps + j * PF_LD + ty * 4);
      const float wv[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const float4 v = *reinterpret_cast<const float4*>(vs + j * DP + tx * 4 + 64 * i);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          o[r][4 * i] = fmaf(wv[r], v.x, o[r][4 * i]);
          o[r][4 * i + 1] = fmaf(wv[r], v.y, o[r][4 * i + 1]);
          o[r][4 * i + 2] = fmaf(wv[r], v.z, o[r][4 * i + 2]);
          o[r][4 * i + 3] = fmaf(wv[r], v.w, o[r][4 * i + 3]);
        }
      }
    }
  }
  uint32_t redo = 0;  // of this warp's rows: 4 (ty & 1) + r
#pragma unroll
  for (int r = 0; r < 4; ++r) {
#pragma unroll
    for (int w = 1; w < 16; w <<= 1) l[r] += __shfl_xor_sync(~0u, l[r], w);
    const int f = t.f0 + ty * 4 + r, tok = fast_div(f, p.group_div);
    const int64_t at = int64_t(t.first + tok) * a.o_stride_t + head[r] * a.o_stride_h;
    float odd = 0.f;
#pragma unroll
    for (int c = 0; c < NI * 4; ++c) {
      const float x = l[r] == 0.f ? 0.f : o[r][c] / l[r];
      const int e = tx * 4 + 64 * (c / 4) + c % 4;
      odd += x * 0.f;
      if (f < last && e < D) store_elem(a.out, a.dtype, at + e, x);
    }
    if (a.lse && tx == 0 && f < last) a.lse[int64_t(t.first + tok) * a.n_q_heads + head[r]] = (m[r] + log2f(l[r])) * kLn2;
    const uint32_t bad = __ballot_sync(~0u, odd != 0.f && l[r] == l[r] && f < last);
    redo |= (bad & 0xFFFFu ? 1u : 0u) << r | (bad >> 16 ? 1u : 0u) << (4 + r);
  }
  if (__syncthreads_or(special)) {
    const int first = t.f0 + (tid >> 5) * 8;  // the warp's rows
    for (int r = 0; r < 8; ++r)
      if (redo >> r & 1) exact_row(p, t, kvh, first + r);
  }
}

// At least one CTA a KV head, for the rows of no request.
int64_t grid_tiles(const PagedParams& p, int size) {
  const int64_t n = most_tiles(p.a.n_rows, p.a.batch, p.group, size);
  return n > 0 ? n : 1;
}

template <class DT, int D>
int launch_mma(const PagedParams& p, cudaStream_t st) {
  auto kern = p.a.softcap > 0.f ? prefill_mma_kernel<DT, D, CAP_ANY> : prefill_mma_kernel<DT, D, CAP_NONE>;
  if (const int rc = allow_smem(reinterpret_cast<const void*>(kern), PmCfg<D>::SMEM, "paged_prefill")) return rc;
  kern<<<dim3(unsigned(grid_tiles(p, PmCfg<D>::ROWS)), p.a.n_kv_heads), PM_THREADS, PmCfg<D>::SMEM, st>>>(p);
  return cuda_status(cudaGetLastError(), "paged_prefill");
}
template <class DT>
int launch_mma_dim(const PagedParams& p, cudaStream_t st) {
  switch (p.a.head_dim) {
    case 64: return launch_mma<DT, 64>(p, st);
    case 128: return launch_mma<DT, 128>(p, st);
    default: return launch_mma<DT, 256>(p, st);
  }
}
template <class DT, int DP, bool VEC>
int launch_fma(const PagedParams& p, cudaStream_t st) {
  if (const int rc = allow_smem(reinterpret_cast<const void*>(prefill_fma_kernel<DT, DP, VEC>), pf_smem<DP>(), "paged_prefill")) return rc;
  prefill_fma_kernel<DT, DP, VEC><<<dim3(unsigned(grid_tiles(p, PF_ROWS)), p.a.n_kv_heads), PF_THREADS, pf_smem<DP>(), st>>>(p);
  return cuda_status(cudaGetLastError(), "paged_prefill");
}
// Tiles of 64 rows from 24 rows a request on (tokens times grouped heads) and 12 rows an SM over all KV heads, tiles of
// four below: they are 16 times as many CTAs, and a CTA is twice as quick.  fp32, 32/8 heads of 128, tiles of 64 / of
// four: 16 requests of 1000 tokens and 2, 4, 8, 16 new ones 207, 329, 335, 340 / 134, 250, 362, 598 us; one of 2000
// tokens and 32, 48, 64, 96, 128 new ones 350, 350, 360, 361, 371 / 199, 219, 419, 429, 633 us.
template <class DT>
int launch_simt(const PagedParams& p, cudaStream_t st) {
  const int D = p.a.head_dim;
  const bool vec = D % 4 == 0 && paged_aligned(p.a);
  if (p.a.n_rows * p.group >= 24 * int64_t(p.a.batch) && p.a.n_rows * p.a.n_q_heads >= 12 * int64_t(num_sms())) {
    if (D <= 64) return vec ? launch_fma<DT, 64, true>(p, st) : launch_fma<DT, 64, false>(p, st);
    if (D <= 128) return vec ? launch_fma<DT, 128, true>(p, st) : launch_fma<DT, 128, false>(p, st);
    return vec ? launch_fma<DT, 256, true>(p, st) : launch_fma<DT, 256, false>(p, st);
  }
  auto go = [&](auto kern) {
    kern<<<dim3(unsigned(grid_tiles(p, PX_ROWS)), p.a.n_kv_heads), PM_THREADS, 0, st>>>(p);
    return cuda_status(cudaGetLastError(), "paged_prefill");
  };
  if (D <= 64) return vec ? go(prefill_simt_kernel<DT, 2, true>) : go(prefill_simt_kernel<DT, 2, false>);
  if (D <= 128) return vec ? go(prefill_simt_kernel<DT, 4, true>) : go(prefill_simt_kernel<DT, 4, false>);
  return vec ? go(prefill_simt_kernel<DT, 8, true>) : go(prefill_simt_kernel<DT, 8, false>);
}

}  // namespace

}  // namespace smaq

extern "C" size_t smaq_paged_prefill_workspace_size(int64_t n_rows, int batch, int n_q_heads, int n_kv_heads, int head_dim, int64_t max_tokens) {
  // only the tensor-core kernel shares walks; the size is the same for every dtype and alignment
  return head_dim == 64 || head_dim == 128 || head_dim == 256 ? smaq::prefill_tc_workspace(n_rows, batch, n_q_heads, n_kv_heads, head_dim, max_tokens) : 0;
}

extern "C" int smaq_paged_prefill(const smaq_paged_args* args, void* stream) {
  using namespace smaq;
  PagedParams p;
  if (const int st = paged_check(args, true, p)) return st;
  const smaq_paged_args& a = p.a;
  if (a.n_rows == 0) return SMAQ_OK;
  if (a.n_kv_heads > 65535) return fail(SMAQ_ERR_UNSUPPORTED, "paged_prefill: %d KV heads above 65535", a.n_kv_heads);
  if (grid_tiles(p, PX_ROWS) >= (int64_t(1) << 31)) return fail(SMAQ_ERR_UNSUPPORTED, "paged_prefill: too many rows");
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (prefill_tc_eligible(a)) return launch_prefill_tc(p, st);
  if (a.dtype != SMAQ_F32 && (a.head_dim == 64 || a.head_dim == 128 || a.head_dim == 256) && paged_aligned(a))
    return a.dtype == SMAQ_BF16 ? launch_mma_dim<BF16>(p, st) : launch_mma_dim<F16>(p, st);
  return a.dtype == SMAQ_F32 ? launch_simt<F32>(p, st) : a.dtype == SMAQ_BF16 ? launch_simt<BF16>(p, st) : launch_simt<F16>(p, st);
}
