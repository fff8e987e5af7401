// Attention of one new token a request over the exact paged cache, split over the cache's length.
//
//   out = sum_j 2^(x_j - m) v_j / sum_j 2^(x_j - m),  x = log2-domain scores, m their running maximum.
//
// Each visible key and value is read once (2 Hkv D L elements a request), 4 G flops an element: HBM-bound,
// so the design is about bytes in flight and an even split.
//
// Split.  A segment is (request, KV head, tile of up to 16 query heads); its visible tokens are cut into
// units of 64, and the units of all segments, in order, are cut into runs of equal cost, one a CTA (two CTAs an
// SM), whatever the lengths.  Each CTA finds its run from seq_lens by itself.  A segment that lies in one
// run is finished there; of the others every CTA leaves (m, sum, accumulator) in slot cta + segment, which is
// distinct because a run's walk raises one of the two at each step, and the join kernel, launched with
// programmatic dependence, adds them in slot order: no atomics, the same result every time.
//
// paged_decode_kernel (bf16 / fp16, head_dim 64 / 128 / 256): four warps, each with its own ring of
// 16-token stages (keys + values, cp.async, 96 KB a CTA and two CTAs an SM in flight), its own softmax
// state and no block-wide barrier until the segment ends.  The page lookups of a stage are made one stage
// before its copies.  Scores by m16n8k16 (rows = query heads of the group, zero rows above it); weights enter
// the second product as hi + lo parts in the cache's type (fp16: scaled by 2^15), which costs tensor time that is idle here
// and keeps 16-bit rounding out of the weights.  Slots past the visible range are filled with zeros by the copy and
// their scores replaced, so what they hold never matters.  64 requests of 1K to 64K tokens at 28/4 heads of 128:
// 315 to 320 us on the device in short runs, 6.4 TB/s; 4 of 128K at 64/8, capped: 337 us, 6.4 TB/s (a plain copy has 6.45).
// In long runs, under the power cap, 334 to 358 and 363 to 393 us a call.
//
// paged_decode_f32_kernel (fp32, head_dim 64 / 128): the same rings; FMA throughout, since tf32 products in three parts
// left 2e-6 in the scores (rounding inside the tensor cores' sums).  33 requests of 100 to 32K tokens, window 4096,
// 12/4 heads of 64: 43 us, of which start and join are 12.
// paged_simt_kernel (other head dims and alignments): 16 groups of eight lanes, one token a group, four query
// rows a tile.
#include <algorithm>

#include "paged.cuh"

namespace smaq {

int paged_check(const smaq_paged_args* args, bool prefill, PagedParams& p) {
  if (!args) return fail(SMAQ_ERR_INVALID, "paged attention: null arguments");
  const smaq_paged_args& a = *args;
  if (a.dtype != SMAQ_F32 && a.dtype != SMAQ_BF16 && a.dtype != SMAQ_F16) return fail(SMAQ_ERR_INVALID, "paged attention: dtype %d", a.dtype);
  if (a.n_kv_heads < 1 || a.n_q_heads < 1 || a.n_q_heads % a.n_kv_heads)
    return fail(SMAQ_ERR_INVALID, "paged attention: head counts %d/%d", a.n_q_heads, a.n_kv_heads);
  if (a.head_dim < 1 || a.head_dim > 256) return fail(SMAQ_ERR_UNSUPPORTED, "paged attention: head_dim %d not in 1..256", a.head_dim);
  if (a.batch < 0 || a.n_rows < 0 || a.page_size < 1 || a.max_blocks < 0 || a.window < 0 || a.n_pages < 0)
    return fail(SMAQ_ERR_INVALID, "paged attention: bad sizes (batch %d, rows %lld, page_size %d, window %d)", a.batch, (long long)a.n_rows,
                a.page_size, a.window);
  if (a.n_rows >= (int64_t(1) << 31) / a.n_q_heads || int64_t(a.batch) * a.n_q_heads >= (int64_t(1) << 31))
    return fail(SMAQ_ERR_UNSUPPORTED, "paged attention: 2^31 rows or more");
  if (!(a.softcap >= 0.f) || !(a.scale == a.scale)) return fail(SMAQ_ERR_INVALID, "paged attention: scale or softcap");
  if (a.table_stride < a.max_blocks) return fail(SMAQ_ERR_INVALID, "paged attention: table stride below its width");
  if (a.n_rows > 0) {
    if (!a.q || !a.out) return fail(SMAQ_ERR_INVALID, "paged attention: null pointer");
    if (a.batch && (!a.seq_lens || (a.max_blocks && a.n_pages && (!a.block_table || !a.k_cache || !a.v_cache))))
      return fail(SMAQ_ERR_INVALID, "paged attention: null pointer");
    if (prefill && !a.cu_query) return fail(SMAQ_ERR_INVALID, "paged attention: null cu_query");
  }
  p.a = a;
  if (a.n_pages == 0) p.a.max_blocks = 0;  // an empty cache: every request reads as empty
  // a window that no request outgrows is none; positions minus it would leave 32 bits
  if (a.window >= std::min(int64_t(a.max_blocks) * a.page_size, int64_t(kLongest))) p.a.window = 0;
  p.group = a.n_q_heads / a.n_kv_heads;
  const float cap = p.a.softcap = a.softcap > 1e30f ? 0.f : a.softcap;  // tanh is the identity at every score: none
  p.scale_log2 = a.scale * kLog2e;
  p.cap_in = cap > 0.f ? 2.0f * kLog2e * a.scale / cap : 0.f;
  p.cap_log2 = cap * kLog2e;
  p.cap_z = cap > kCapNear ? a.scale / cap : 0.f;
  p.page_div = make_fastdiv(a.page_size);
  p.group_div = make_fastdiv(p.group);
  return SMAQ_OK;
}

bool paged_aligned(const smaq_paged_args& a) {
  const int64_t e = a.dtype == SMAQ_F32 ? 4 : 2;
  const uintptr_t ptrs = reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.k_cache) | reinterpret_cast<uintptr_t>(a.v_cache) |
                         reinterpret_cast<uintptr_t>(a.out);
  const int64_t strides = a.q_stride_t | a.q_stride_h | a.c_stride_page | a.c_stride_slot | a.c_stride_h | a.o_stride_t | a.o_stride_h;
  return ptrs % 16 == 0 && (strides * e) % 16 == 0;
}

namespace {

constexpr int PD_UNIT = 64;    // tokens a unit
constexpr int PD_THREADS = 128;

struct DecodeParamsX {
  PagedParams p;
  int tiles;      // tiles of query heads a KV head
  int rows;       // query heads a tile, at most
  int segs;       // n_kv_heads * tiles
  int grid;
  float* slots;   // [grid + batch * segs][rows][head_dim + 2]
};

struct Visible {
  int lo, hi, units;
};
__device__ __forceinline__ Visible visible(const PagedParams& p, int b) {
  Visible v;
  v.hi = paged_len(p, b);
  v.lo = p.a.window > 0 && v.hi > p.a.window ? v.hi - p.a.window : 0;
  v.units = (v.hi - v.lo + PD_UNIT - 1) / PD_UNIT;
  return v;
}

// Sum over the block (PD_THREADS threads) of one int64 a thread, and the sum before this thread.
__device__ __forceinline__ int64_t block_prefix(int64_t v, int64_t* warp_sums, int64_t& before) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  int64_t x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t u = __shfl_up_sync(~0u, x, o);
    if (lane >= o) x += u;
  }
  __syncthreads();
  if (lane == 31) warp_sums[w] = x;
  __syncthreads();
  int64_t total = 0, base = 0;
#pragma unroll
  for (int i = 0; i < PD_THREADS / 32; ++i) {
    if (i < w) base += warp_sums[i];
    total += warp_sums[i];
  }
  before = base + x - v;
  return total;
}

// Walks the units of a run in order: request, segment of it, unit of the segment.
struct Walk {
  int b, s, t;
  Visible v;
  // to the next unit; the caller knows that one exists
  __device__ __forceinline__ void next(const DecodeParamsX& d) {
    if (++t < v.units) return;
    t = 0;
    if (++s < d.segs) return;
    s = 0;
    do {
      ++b;
      v = visible(d.p, b);
    } while (v.units == 0 && b + 1 < d.p.a.batch);
  }
};

// Runs are equal in cost: a unit costs 1, and beginning a segment (its queries, and joining the warps at its end) as
// much as PD_START units of a CTA among others.  Without that, CTAs that met many short segments ended 10 us after the
// others in a ragged windowed batch.  The cost of a request's segments and how many requests have any, packed:
constexpr int PD_START = 1, PD_PACK = 24;  // batch < 2^24
__device__ __forceinline__ int64_t packed_cost(const DecodeParamsX& d, int b) {
  const int units = b < d.p.a.batch ? visible(d.p, b).units : 0;
  return units ? (int64_t(units + PD_START) * d.segs << PD_PACK) + 1 : 0;
}
// Run of CTA c: costs [first(c), first(c + 1)).  With a total below the number of CTAs, the first ones get 1
// each, so that no CTA between those of a segment's first and last unit is without a unit of it.
__device__ __forceinline__ int64_t run_first(int64_t c, int64_t total, int grid) {
  return total < grid ? min(c, total) : c * total / grid;
}
// The CTA that has cost position u.
__device__ __forceinline__ int run_of(int64_t u, int64_t total, int grid) {
  return total < grid ? int(u) : int(((u + 1) * grid - 1) / total);
}

struct Spot {
  int b, s, t;    // a unit
  int64_t index;  // its number among all units
};
struct RunShared {
  int64_t warp_sums[PD_THREADS / 32];
  Spot spot[2];
};

// The CTA's run: its first unit and the number of its units.
__device__ __forceinline__ int find_run(const DecodeParamsX& d, RunShared& sh, Walk& at) {
  const int B = d.p.a.batch;
  int64_t sum = 0, mine = 0, before = 0;
  for (int b0 = 0; b0 < B; b0 += PD_THREADS) {
    mine = packed_cost(d, b0 + threadIdx.x);
    sum += block_prefix(mine, sh.warp_sums, before);
  }
  constexpr int64_t COUNT = (int64_t(1) << PD_PACK) - 1;
  const int64_t total = sum >> PD_PACK;
  const int64_t ends[2] = {run_first(blockIdx.x, total, d.grid), run_first(int64_t(blockIdx.x) + 1, total, d.grid)};
  if (ends[0] == ends[1]) return 0;
  if (threadIdx.x == 0) sh.spot[1].index = total - (sum & COUNT) * PD_START * d.segs;  // the end of all
  __syncthreads();
  int64_t base = 0;
  for (int b0 = 0; b0 < B && (base >> PD_PACK) <= ends[1]; b0 += PD_THREADS) {
    int64_t chunk = sum;
    if (B > PD_THREADS) {
      mine = packed_cost(d, b0 + threadIdx.x);
      chunk = block_prefix(mine, sh.warp_sums, before);
    }
    const int64_t from = base + before, cost = from >> PD_PACK;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int64_t into = ends[e] - cost;
      if (mine && into >= 0 && into < mine >> PD_PACK) {
        const int per = int((mine >> PD_PACK) / d.segs), s = int(into / per), t = max(int(into - int64_t(s) * per) - PD_START, 0);
        const int units = per - PD_START;
        sh.spot[e] = {b0 + int(threadIdx.x), s, t, cost - (from & COUNT) * PD_START * d.segs + int64_t(s) * units + t};
      }
    }
    base += chunk;
  }
  __syncthreads();
  at.b = sh.spot[0].b;
  at.s = sh.spot[0].s;
  at.t = sh.spot[0].t;
  at.v = visible(d.p, at.b);
  return int(sh.spot[1].index - sh.spot[0].index);
}

// Rows of requests that see nothing.
__device__ __forceinline__ void write_empty(const DecodeParamsX& d) {
  const smaq_paged_args& a = d.p.a;
  for (int b = blockIdx.x; b < a.batch; b += gridDim.x) {
    if (visible(d.p, b).units) continue;
    for (int i = threadIdx.x; i < a.n_q_heads * a.head_dim; i += blockDim.x)
      store_elem(a.out, a.dtype, b * a.o_stride_t + (i / a.head_dim) * a.o_stride_h + i % a.head_dim, 0.f);
    if (a.lse)
      for (int h = threadIdx.x; h < a.n_q_heads; h += blockDim.x) a.lse[int64_t(b) * a.n_q_heads + h] = -INFINITY;
  }
}

// Accumulator of one row over tokens [lo, hi) for a known maximum m, by one warp in 32 bits, into acc[0, D).
// The hi + lo parts of a weight times an infinite value give NaN where their sum gives the infinity; a row that
// comes out without a finite value is redone here, token by token: such values are rare, and a call that meets one is slow
// (4 requests of 64K tokens at 32/8 heads, one infinity: 68 ms instead of 0.26).
template <int CAP>
__device__ __noinline__ void redo_row(const PagedParams& p, int b, int h, int lo, int hi, int last, float m, float* acc) {
  const smaq_paged_args& a = p.a;
  const int lane = threadIdx.x & 31, D = a.head_dim;
  const int32_t* table = a.block_table + b * a.table_stride;
  const float slope = a.slopes ? a.slopes[h] * kLog2e : 0.f;
  float o[8] = {};
  for (int j = lo; j < hi; ++j) {
    const int64_t off = token_offset(p, table, j) + (h / p.group) * a.c_stride_h;
    float x = 0.f;
    for (int e = lane; e < D; e += 32)
      x = fmaf(load_elem(a.q, a.dtype, b * a.q_stride_t + h * a.q_stride_h + e), load_elem(a.k_cache, a.dtype, off + e), x);
    const float w = ex2(score_log2<CAP>(warp_sum(x), p) - slope * float(last - j) - m);
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (lane + 32 * k < D) o[k] += w * load_elem(a.v_cache, a.dtype, off + lane + 32 * k);
  }
#pragma unroll
  for (int k = 0; k < 8; ++k)
    if (lane + 32 * k < D) acc[lane + 32 * k] = o[k];
}

// Stages of 16 tokens, keys then values, of ROW bytes a token: a warp's ring.
template <int ROW>
struct Stages {
  static constexpr int BYTES = 16 * ROW * 2;
  static constexpr int N = ROW == 128 ? 6 : 3;
  static constexpr int CTAS = ROW == 512 ? 1 : 2;                // an SM
};

// A warp's copies: the walk runs ahead of the computing one by N - 1 units, its page lookups by one more.
template <class T, int ROW>
struct Feed {
  using S = Stages<ROW>;
  static constexpr int CH = ROW / 16;  // 16-byte chunks a token; chunk c of row r lies at c ^ (r % 8)
  Walk in;
  int count, looked = 0, issued = 0;
  const uint8_t* row = nullptr;  // this lane's chunk of the keys of token (lane & 15) of the unit looked up last
  uint32_t visible_rows = 0;     // bit r: token r of it is visible, from this lane's first row on
  uint8_t* ring;

  __device__ __forceinline__ void start(const DecodeParamsX& d, const Walk& first, int units, uint8_t* at) {
    in = first;
    count = units;
    ring = at;
    // the first stages' lookups side by side: one after the other they took 3 us before the first copy
    const uint8_t* rows[S::N];
    uint32_t seen[S::N];
#pragma unroll
    for (int i = 0; i < S::N; ++i) {
      look_up(d);
      rows[i] = row;
      seen[i] = visible_rows;
    }
#pragma unroll
    for (int i = 0; i < S::N; ++i) {
      row = rows[i];
      visible_rows = seen[i];
      if (i + 1 < S::N) issue(d);
    }
  }
  __device__ __forceinline__ void look_up(const DecodeParamsX& d) {
    if (looked >= count) return;
    if (looked) in.next(d);
    ++looked;
    const int lane = threadIdx.x & 31, j0 = in.v.lo + in.t * PD_UNIT + (threadIdx.x >> 5) * 16, j = j0 + (lane & 15);
    const int n = min(max(in.v.hi - j0, 0), 16);
    int64_t off = 0;
    if (j < in.v.hi)
      off = token_offset(d.p, d.p.a.block_table + in.b * d.p.a.table_stride, j) + int64_t(in.s / d.tiles) * d.p.a.c_stride_h;
    row = static_cast<const uint8_t*>(d.p.a.k_cache) + off * int64_t(sizeof(T));
    visible_rows = ((1u << n) - 1u) >> (lane / CH);
  }
  __device__ __forceinline__ void issue(const DecodeParamsX& d) {
    if (issued < count) {
      const int lane = threadIdx.x & 31;
      // a step is 32 / CH rows; the swizzle of its first row is a constant, that of the lane's row within it is not
      constexpr int PER = 32 / CH;
      const int mine = lane / CH, ch = lane % CH;
      const uint32_t st = smem_u32(ring + (issued % S::N) * S::BYTES);
      const uint32_t lane_dst = uint32_t(mine * ROW + ((ch ^ mine) << 4));
      const int64_t to_values = static_cast<const uint8_t*>(d.p.a.v_cache) - static_cast<const uint8_t*>(d.p.a.k_cache) + ch * 16;
#pragma unroll
      for (int i = 0; i < 16 / PER; ++i) {
        const uint8_t* from = reinterpret_cast<const uint8_t*>(__shfl_sync(~0u, reinterpret_cast<uint64_t>(row), i * PER + mine));
        const uint32_t at = st + uint32_t(i * PER * ROW) + (lane_dst ^ uint32_t((i * PER & 7) << 4));
        const uint32_t n = (visible_rows >> (i * PER) & 1u) << 4;
        cp_async16(at, from + ch * 16, n);
        cp_async16(at + 16 * ROW, from + to_values, n);
      }
      ++issued;
    }
    cp_async_commit();
  }
  // Stage of unit i, whole; the copies of unit i + N - 1 go into the stage of the unit before it.
  __device__ __forceinline__ uint8_t* stage(const DecodeParamsX& d, int i) {
    cp_async_wait<S::N - 2>();
    __syncwarp();
    issue(d);
    look_up(d);
    return ring + (i % S::N) * S::BYTES;
  }
};

template <int D>
struct Cfg {
  using S = Stages<2 * D>;
  static constexpr int LD = D + 2;                               // floats of a merge row: accumulator, m, sum
  static constexpr int SMEM = 4 * S::N * S::BYTES + 2 * 16 * LD * 4;
};

template <class DT, int D, int CAP>
__global__ void __launch_bounds__(PD_THREADS, Stages<2 * D>::CTAS) paged_decode_kernel(const __grid_constant__ DecodeParamsX d) {
  using T = typename DT::T;
  constexpr int LD = Cfg<D>::LD;
  constexpr int KS = D / 16;        // contraction steps of the scores
  constexpr int NT = D / 8;         // output column tiles
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ RunShared run;
  const PagedParams& p = d.p;
  const smaq_paged_args& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_launch_dependents();
  Walk at;
  const int count = find_run(d, run, at);

  using S = Stages<2 * D>;
  float* merge = reinterpret_cast<float*>(smem + 4 * S::N * S::BYTES);
  Feed<T, 2 * D> feed;
  if (count > 0) feed.start(d, at, count, smem + warp * S::N * S::BYTES);
  write_empty(d);  // behind the first copies
  if (count <= 0) return;

  // ---- compute
  uint32_t qf[KS][4];
  float o[NT][4];
  float m0, m1, l0, l1;  // rows lane / 4 and lane / 4 + 8
  float slope0 = 0.f, slope1 = 0.f;
  bool fresh = true;
  int from = at.t;  // first unit of the segment in this run
#pragma unroll 1
  for (int i = 0; i < count; ++i) {
    if (fresh) {
      fresh = false;
      m0 = m1 = -INFINITY;
      l0 = l1 = 0.f;
#pragma unroll
      for (int n = 0; n < NT; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
      const int kvh = at.s / d.tiles, tile = at.s - kvh * d.tiles;
      const int first = kvh * p.group + tile * 16, rows = min(16, p.group - tile * 16);
      const int r0 = lane >> 2, r1 = r0 + 8;
      const T* q = static_cast<const T*>(a.q) + at.b * a.q_stride_t + 2 * (lane & 3);
      const T* q0 = q + (first + r0) * a.q_stride_h;
      const T* q1 = q + (first + r1) * a.q_stride_h;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        qf[k][0] = r0 < rows ? __ldg(reinterpret_cast<const uint32_t*>(q0 + k * 16)) : 0u;
        qf[k][1] = r1 < rows ? __ldg(reinterpret_cast<const uint32_t*>(q1 + k * 16)) : 0u;
        qf[k][2] = r0 < rows ? __ldg(reinterpret_cast<const uint32_t*>(q0 + k * 16 + 8)) : 0u;
        qf[k][3] = r1 < rows ? __ldg(reinterpret_cast<const uint32_t*>(q1 + k * 16 + 8)) : 0u;
      }
      if (a.slopes) {
        slope0 = r0 < rows ? a.slopes[first + r0] * kLog2e : 0.f;
        slope1 = r1 < rows ? a.slopes[first + r1] * kLog2e : 0.f;
      }
    }
    const uint32_t ks = smem_u32(feed.stage(d, i)), vs = ks + 16 * D * 2;
    const int j0 = at.v.lo + at.t * PD_UNIT + warp * 16;
    if (j0 < at.v.hi) {
      float c[2][4] = {};
      // keys: tokens 0-7 / 8-15 (matrix pairs), channels 16k .. 16k + 15
      const int kr = (lane & 7) + ((lane >> 4) << 3), kc = (lane >> 3) & 1;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        uint32_t b[4];
        ldmatrix4(b, ks + uint32_t(kr * D * 2 + (((2 * k + kc) ^ (kr & 7)) << 4)));
        mma_16816<DT>(c[0], qf[k], b[0], b[1]);
        mma_16816<DT>(c[1], qf[k], b[2], b[3]);
      }
      float mx0 = -INFINITY, mx1 = -INFINITY;
      const int last = at.v.hi - 1;
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int j = j0 + n * 8 + 2 * (lane & 3) + e;
          const float gap = float(last - j);
          float x0 = score_log2<CAP>(c[n][e], p) - slope0 * gap, x1 = score_log2<CAP>(c[n][2 + e], p) - slope1 * gap;
          c[n][e] = x0 = j <= last ? x0 : -INFINITY;
          c[n][2 + e] = x1 = j <= last ? x1 : -INFINITY;
          mx0 = fmaxf(mx0, x0);
          mx1 = fmaxf(mx1, x1);
        }
#pragma unroll
      for (int w = 1; w < 4; w <<= 1) {
        mx0 = fmaxf(mx0, __shfl_xor_sync(~0u, mx0, w));
        mx1 = fmaxf(mx1, __shfl_xor_sync(~0u, mx1, w));
      }
      mx0 -= kUp<DT>;  // m lies that much below the maximum from here on, in the slots too
      mx1 -= kUp<DT>;
      if (__any_sync(~0u, mx0 > m0 || mx1 > m1)) {
        const float n0 = fmaxf(m0, mx0), n1 = fmaxf(m1, mx1);
        const float f0 = m0 == -INFINITY ? 0.f : ex2(m0 - n0), f1 = m1 == -INFINITY ? 0.f : ex2(m1 - n1);
        m0 = n0;
        m1 = n1;
        l0 *= f0;
        l1 *= f1;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          o[n][0] *= f0;
          o[n][1] *= f0;
          o[n][2] *= f1;
          o[n][3] *= f1;
        }
      }
      const float b0 = m0 == -INFINITY ? 0.f : m0, b1 = m1 == -INFINITY ? 0.f : m1;
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const float p00 = ex2(c[n][0] - b0), p01 = ex2(c[n][1] - b0), p10 = ex2(c[n][2] - b1), p11 = ex2(c[n][3] - b1);
        l0 += p00 + p01;
        l1 += p10 + p11;
        hi[2 * n] = pack2<DT>(p00, p01);
        hi[2 * n + 1] = pack2<DT>(p10, p11);
        const float2 h0 = unpack2<DT>(hi[2 * n]), h1 = unpack2<DT>(hi[2 * n + 1]);
        lo[2 * n] = pack2<DT>(p00 - h0.x, p01 - h0.y);
        lo[2 * n + 1] = pack2<DT>(p10 - h1.x, p11 - h1.y);
      }
      // values: tokens 0-7 / 8-15, channels 16n .. 16n + 15, transposed
      const int vr = (lane & 7) + (((lane >> 3) & 1) << 3), vc = lane >> 4;
#pragma unroll
      for (int n = 0; n < NT / 2; ++n) {
        uint32_t b[4];
        ldmatrix4_trans(b, vs + uint32_t(vr * D * 2 + (((2 * n + vc) ^ (vr & 7)) << 4)));
        mma_16816<DT>(o[2 * n], hi, b[0], b[1]);
        mma_16816<DT>(o[2 * n + 1], hi, b[2], b[3]);
        mma_16816<DT>(o[2 * n], lo, b[0], b[1]);
        mma_16816<DT>(o[2 * n + 1], lo, b[2], b[3]);
      }
    }

    const bool ends = at.t + 1 == at.v.units;
    if (ends || i + 1 == count) {
      // ---- the four warps' states into one: 2, 3 -> 0, 1; 1 -> 0
      l0 += __shfl_xor_sync(~0u, l0, 1);
      l1 += __shfl_xor_sync(~0u, l1, 1);
      l0 += __shfl_xor_sync(~0u, l0, 2);
      l1 += __shfl_xor_sync(~0u, l1, 2);
      const int r0 = lane >> 2, r1 = r0 + 8, col = 2 * (lane & 3);
      auto put = [&](float* dst) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          *reinterpret_cast<float2*>(dst + r0 * LD + n * 8 + col) = make_float2(o[n][0], o[n][1]);
          *reinterpret_cast<float2*>(dst + r1 * LD + n * 8 + col) = make_float2(o[n][2], o[n][3]);
        }
        if ((lane & 3) == 0) {
          *reinterpret_cast<float2*>(dst + r0 * LD + D) = make_float2(m0, l0);
          *reinterpret_cast<float2*>(dst + r1 * LD + D) = make_float2(m1, l1);
        }
      };
      auto add = [&](const float* src) {
        const float2 s0 = *reinterpret_cast<const float2*>(src + r0 * LD + D), s1 = *reinterpret_cast<const float2*>(src + r1 * LD + D);
        const float n0 = fmaxf(m0, s0.x), n1 = fmaxf(m1, s1.x);
        const float z0 = n0 == -INFINITY ? 0.f : n0, z1 = n1 == -INFINITY ? 0.f : n1;
        const float f0 = ex2(m0 - z0), f1 = ex2(m1 - z1), g0 = ex2(s0.x - z0), g1 = ex2(s1.x - z1);
        m0 = n0;
        m1 = n1;
        l0 = l0 * f0 + s0.y * g0;
        l1 = l1 * f1 + s1.y * g1;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const float2 x0 = *reinterpret_cast<const float2*>(src + r0 * LD + n * 8 + col);
          const float2 x1 = *reinterpret_cast<const float2*>(src + r1 * LD + n * 8 + col);
          o[n][0] = o[n][0] * f0 + x0.x * g0;
          o[n][1] = o[n][1] * f0 + x0.y * g0;
          o[n][2] = o[n][2] * f1 + x1.x * g1;
          o[n][3] = o[n][3] * f1 + x1.y * g1;
        }
      };
      __syncthreads();  // the merge rows of the segment before are read
      if (warp >= 2) put(merge + (warp - 2) * 16 * LD);
      __syncthreads();
      if (warp < 2) add(merge + warp * 16 * LD);
      if (warp == 1) {
        __syncwarp();  // all lanes have read the rows that the next lines overwrite
        put(merge + 16 * LD);
      }
      __syncthreads();
      if (warp == 0) {
        add(merge + 16 * LD);
        const int kvh = at.s / d.tiles, tile = at.s - kvh * d.tiles;
        const int first = kvh * p.group + tile * 16, rows = min(16, p.group - tile * 16);
        float odd0 = 0.f, odd1 = 0.f;  // NaN where the accumulator is not finite and the weights are
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          odd0 += (o[n][0] + o[n][1]) * 0.f;
          odd1 += (o[n][2] + o[n][3]) * 0.f;
        }
        const uint32_t redo0 = __ballot_sync(~0u, odd0 != 0.f && l0 * 0.f == 0.f), redo1 = __ballot_sync(~0u, odd1 != 0.f && l1 * 0.f == 0.f);
        if (redo0 | redo1) {
          for (int r = 0; r < rows; ++r) {
            if (!((r < 8 ? redo0 : redo1) >> (4 * (r & 7)) & 15u)) continue;
            const float m = __shfl_sync(~0u, r < 8 ? m0 : m1, 4 * (r & 7));
            redo_row<CAP>(p, at.b, first + r, at.v.lo + from * PD_UNIT, min(at.v.hi, at.v.lo + (at.t + 1) * PD_UNIT), at.v.hi - 1, m, merge);
            __syncwarp();
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const float2 x = *reinterpret_cast<const float2*>(merge + n * 8 + col);
              const int e = r < 8 ? 0 : 2;
              if (r == (e ? r1 : r0)) {  // finite elements stay as they are
                if (!isfinite(e ? o[n][2] : o[n][0])) (e ? o[n][2] : o[n][0]) = x.x;
                if (!isfinite(e ? o[n][3] : o[n][1])) (e ? o[n][3] : o[n][1]) = x.y;
              }
            }
            __syncwarp();
          }
        }
        if (ends && from == 0) {
          const float i0 = l0 > 0.f ? 1.0f / l0 : (l0 == 0.f ? 0.f : l0), i1 = l1 > 0.f ? 1.0f / l1 : (l1 == 0.f ? 0.f : l1);
          T* out = static_cast<T*>(a.out) + at.b * a.o_stride_t + col;
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            if (r0 < rows) *reinterpret_cast<uint32_t*>(out + (first + r0) * a.o_stride_h + n * 8) = pack2<DT>(o[n][0] * i0, o[n][1] * i0);
            if (r1 < rows) *reinterpret_cast<uint32_t*>(out + (first + r1) * a.o_stride_h + n * 8) = pack2<DT>(o[n][2] * i1, o[n][3] * i1);
          }
          if (a.lse && (lane & 3) == 0) {
            float* lse = a.lse + int64_t(at.b) * a.n_q_heads + first;
            if (r0 < rows) lse[r0] = (m0 + log2f(l0)) * kLn2;
            if (r1 < rows) lse[r1] = (m1 + log2f(l1)) * kLn2;
          }
        } else {
          float* slot = d.slots + (int64_t(blockIdx.x) + int64_t(at.b) * d.segs + at.s) * d.rows * LD;
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            if (r0 < rows) *reinterpret_cast<float2*>(slot + r0 * LD + n * 8 + col) = make_float2(o[n][0], o[n][1]);
            if (r1 < rows) *reinterpret_cast<float2*>(slot + r1 * LD + n * 8 + col) = make_float2(o[n][2], o[n][3]);
          }
          if ((lane & 3) == 0) {
            if (r0 < rows) *reinterpret_cast<float2*>(slot + r0 * LD + D) = make_float2(m0, l0);
            if (r1 < rows) *reinterpret_cast<float2*>(slot + r1 * LD + D) = make_float2(m1, l1);
          }
        }
      }
      fresh = true;
      from = 0;
    }
    if (i + 1 < count) at.next(d);
  }
}

// ---------------------------------------------------------------- fp32
// R query heads a tile.  Scores: lane = (half of the channels, token), so that a 16-token stage takes one exchange a
// row; weighted values: lane = D / 32 channels, the weights broadcast from shared memory.
template <int D, int R>
struct FCfg {
  using S = Stages<4 * D>;
  static constexpr int QH = D / 2 + 4;                 // floats of half a query row: the halves start four banks apart
  static constexpr int AREA = R * 2 * QH;              // a warp's query rows, at the end of a segment its accumulators
  static constexpr int SMEM = 4 * (S::N * S::BYTES + (AREA + 16 * R) * 4);
};

template <int D, int R, bool CAP>
__global__ void __launch_bounds__(PD_THREADS, Stages<4 * D>::CTAS) paged_decode_f32_kernel(const __grid_constant__ DecodeParamsX d) {
  using Q = FCfg<D, R>;
  using S = Stages<4 * D>;
  constexpr int E = D / 32, LD = D + 2;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ RunShared run;
  const PagedParams& p = d.p;
  const smaq_paged_args& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_launch_dependents();
  Walk at;
  const int count = find_run(d, run, at);
  Feed<float, 4 * D> feed;
  if (count > 0) feed.start(d, at, count, smem + warp * S::N * S::BYTES);
  write_empty(d);  // behind the first copies
  if (count <= 0) return;
  float* areas = reinterpret_cast<float*>(smem + 4 * S::N * S::BYTES);
  float *mine = areas + warp * Q::AREA, *ps = areas + 4 * Q::AREA + warp * 16 * R;

  const int tok = lane & 15, half = lane >> 4;
  float o[R][E], m[R], l[R], slope[R];
  bool fresh = true;
  int from = at.t;
#pragma unroll 1
  for (int i = 0; i < count; ++i) {
    const int kvh = at.s / d.tiles, tile = at.s - kvh * d.tiles;
    const int first = kvh * p.group + tile * R, rows = min(R, p.group - tile * R);
    if (fresh) {
      fresh = false;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        m[r] = -INFINITY;
        l[r] = 0.f;
        slope[r] = a.slopes && r < rows ? a.slopes[first + r] * kLog2e : 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) o[r][e] = 0.f;
      }
      for (int k = lane; k < R * D; k += 32) {
        const int r = k / D, e = k % D;
        mine[(2 * r + e / (D / 2)) * Q::QH + e % (D / 2)] =
            r < rows ? static_cast<const float*>(a.q)[at.b * a.q_stride_t + (first + r) * a.q_stride_h + e] : 0.f;
      }
    }
    const uint8_t* ks = feed.stage(d, i);  // waits for the whole warp: the query rows are there too
    const uint8_t* vs = ks + 16 * 4 * D;
    const int j0 = at.v.lo + at.t * PD_UNIT + warp * 16, last = at.v.hi - 1;
    if (j0 <= last) {
      float x[R];
#pragma unroll
      for (int r = 0; r < R; ++r) x[r] = 0.f;
#pragma unroll
      for (int c = 0; c < D / 8; ++c) {
        const float4 k = *reinterpret_cast<const float4*>(ks + tok * 4 * D + (((half * (D / 8) + c) ^ (tok & 7)) << 4));
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float4 q = *reinterpret_cast<const float4*>(mine + (2 * r + half) * Q::QH + 4 * c);
          x[r] = fmaf(q.x, k.x, fmaf(q.y, k.y, fmaf(q.z, k.z, fmaf(q.w, k.w, x[r]))));
        }
      }
      const int j = j0 + tok;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float y = x[r] + __shfl_xor_sync(~0u, x[r], 16);
        if constexpr (CAP) y = a.softcap * kLog2e * tanhf(y * a.scale / a.softcap);
        else y *= p.scale_log2;
        y = j <= last ? y - slope[r] * float(last - j) : -INFINITY;
        if (__any_sync(~0u, y > m[r])) {
          float n = fmaxf(m[r], y);
#pragma unroll
          for (int w = 8; w > 0; w >>= 1) n = fmaxf(n, __shfl_xor_sync(~0u, n, w));
          const float f = m[r] == -INFINITY ? 0.f : ex2(m[r] - n);
          m[r] = n;
          l[r] *= f;
#pragma unroll
          for (int e = 0; e < E; ++e) o[r][e] *= f;
        }
        x[r] = ex2(y - (m[r] == -INFINITY ? 0.f : m[r]));
        l[r] += x[r];
      }
      if (half == 0) {
#pragma unroll
        for (int r = 0; r < R; r += 4) *reinterpret_cast<float4*>(ps + tok * R + r) = make_float4(x[r], x[r + 1], x[r + 2], x[r + 3]);
      }
      __syncwarp();
#pragma unroll
      for (int t = 0; t < 16; ++t) {
        float v[E];
        const uint8_t* row = vs + t * 4 * D;
        if constexpr (E == 2) {
          const float2 u = *reinterpret_cast<const float2*>(row + (((lane >> 1) ^ (t & 7)) << 4) + (lane & 1) * 8);
          v[0] = u.x;
          v[1] = u.y;
        } else {
          const float4 u = *reinterpret_cast<const float4*>(row + ((lane ^ (t & 7)) << 4));
          v[0] = u.x;
          v[1] = u.y;
          v[2] = u.z;
          v[3] = u.w;
        }
#pragma unroll
        for (int r = 0; r < R; r += 4) {
          const float4 w = *reinterpret_cast<const float4*>(ps + t * R + r);
#pragma unroll
          for (int e = 0; e < E; ++e) {
            o[r][e] = fmaf(w.x, v[e], o[r][e]);
            o[r + 1][e] = fmaf(w.y, v[e], o[r + 1][e]);
            o[r + 2][e] = fmaf(w.z, v[e], o[r + 2][e]);
            o[r + 3][e] = fmaf(w.w, v[e], o[r + 3][e]);
          }
        }
      }
      __syncwarp();  // before the weights of the next stage
    }

    const bool ends = at.t + 1 == at.v.units;
    if (ends || i + 1 == count) {
      // ---- the four warps' states into one
#pragma unroll
      for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int w = 8; w > 0; w >>= 1) l[r] += __shfl_xor_sync(~0u, l[r], w);
#pragma unroll
        for (int e = 0; e < E; ++e) mine[r * LD + E * lane + e] = o[r][e];
        if (lane == 0) {
          mine[r * LD + D] = m[r];
          mine[r * LD + D + 1] = l[r];
        }
      }
      __syncthreads();
      const bool all = ends && from == 0;
      float* slot = d.slots + (int64_t(blockIdx.x) + int64_t(at.b) * d.segs + at.s) * d.rows * LD;
      for (int k = threadIdx.x; k < rows * D; k += PD_THREADS) {
        const int r = k / D, e = k - r * D;
        float mm = -INFINITY;
#pragma unroll
        for (int w = 0; w < 4; ++w) mm = fmaxf(mm, areas[w * Q::AREA + r * LD + D]);
        const float z = mm == -INFINITY ? 0.f : mm;
        float x = 0.f, sum = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          // a warp without tokens holds zeros; one whose scores are NaN has no maximum either, and its sum stays NaN times zero
          const float f = ex2(areas[w * Q::AREA + r * LD + D] - z);
          x += f * areas[w * Q::AREA + r * LD + e];
          sum += f * areas[w * Q::AREA + r * LD + D + 1];
        }
        if (all) {
          static_cast<float*>(a.out)[at.b * a.o_stride_t + (first + r) * a.o_stride_h + e] = sum == 0.f ? 0.f : x / sum;
          if (a.lse && e == 0) a.lse[int64_t(at.b) * a.n_q_heads + first + r] = (mm + log2f(sum)) * kLn2;
        } else {
          slot[r * LD + e] = x;
          if (e == 0) {
            slot[r * LD + D] = mm;
            slot[r * LD + D + 1] = sum;
          }
        }
      }
      __syncthreads();  // before the areas hold the next segment's queries
      fresh = true;
      from = 0;
    }
    if (i + 1 < count) at.next(d);
  }
}

// ---------------------------------------------------------------- other types, head dims and alignments
constexpr int PS_ROWS = 4;  // query heads a tile

// NI vectors of four elements a lane, element 4 * (l + 8 * i); VEC: whole aligned vectors.
template <class DT, int NI, bool VEC>
__device__ __forceinline__ void load_row(const typename DT::T* row, int l, int D, float (&x)[NI][4]) {
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int e = 4 * (l + 8 * i);
    if constexpr (VEC) {
      if (e < D) load_vec<DT, 4>(row + e, x[i]);
      else x[i][0] = x[i][1] = x[i][2] = x[i][3] = 0.f;
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) x[i][k] = e + k < D ? to_f(row[e + k]) : 0.f;
    }
  }
}

template <class DT, int NI, bool VEC>
__global__ void __launch_bounds__(PD_THREADS) paged_simt_kernel(const __grid_constant__ DecodeParamsX d) {
  using T = typename DT::T;
  constexpr int GROUPS = PD_THREADS / 8;
  __shared__ RunShared run;
  __shared__ __align__(16) float qs[PS_ROWS][32 * NI];
  __shared__ float acc[PD_THREADS / 32][PS_ROWS][32 * NI + 2];
  const PagedParams& p = d.p;
  const smaq_paged_args& a = p.a;
  const int D = a.head_dim, LD = D + 2, l = threadIdx.x & 7, grp = threadIdx.x >> 3, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  pdl_launch_dependents();
  write_empty(d);
  Walk at;
  int left = find_run(d, run, at);
  if (left <= 0) return;
  while (left > 0) {
    const int n = min(left, at.v.units - at.t);  // units of this segment in the run
    const int kvh = at.s / d.tiles, tile = at.s - kvh * d.tiles;
    const int first = kvh * p.group + tile * PS_ROWS, rows = min(PS_ROWS, p.group - tile * PS_ROWS);
    __syncthreads();
    for (int i = threadIdx.x; i < PS_ROWS * 32 * NI; i += PD_THREADS) {
      const int r = i / (32 * NI), e = i % (32 * NI);
      qs[r][e] = r < rows && e < D ? load_elem(a.q, a.dtype, at.b * a.q_stride_t + (first + r) * a.q_stride_h + e) : 0.f;
    }
    __syncthreads();
    float o[PS_ROWS][NI][4] = {}, m[PS_ROWS], s[PS_ROWS], slope[PS_ROWS];
#pragma unroll
    for (int r = 0; r < PS_ROWS; ++r) {
      m[r] = -INFINITY;
      s[r] = 0.f;
      slope[r] = a.slopes && r < rows ? a.slopes[first + r] : 0.f;
    }
    const int lo = at.v.lo + at.t * PD_UNIT, hi = min(at.v.hi, lo + n * PD_UNIT), last = at.v.hi - 1;
    const int32_t* table = a.block_table + at.b * a.table_stride;
    const T* kc = static_cast<const T*>(a.k_cache) + kvh * a.c_stride_h;
    const T* vc = static_cast<const T*>(a.v_cache) + kvh * a.c_stride_h;
    // keys and values a step ahead where registers allow, addresses two
    constexpr bool AHEAD = NI <= 4;
    float nk[NI][4], nv[NI][4];
    auto offset = [&](int j) { return j < hi ? token_offset(p, table, j) : int64_t(-1); };
    auto fetch = [&](int64_t off) {
      if (off >= 0) {
        load_row<DT, NI, VEC>(kc + off, l, D, nk);
        load_row<DT, NI, VEC>(vc + off, l, D, nv);
        return;
      }
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) nk[i][e] = nv[i][e] = 0.f;
    };
    int64_t next = offset(lo + grp);
    if (AHEAD) {
      fetch(next);
      next = offset(lo + GROUPS + grp);
    }
    for (int j0 = lo; j0 < hi; j0 += GROUPS) {  // the same number of steps for every group: whole warps shuffle
      const int j = j0 + grp;
      const bool seen = j < hi;
      float k[NI][4], v[NI][4];
      if (!AHEAD) fetch(next);
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          k[i][e] = nk[i][e];
          v[i][e] = nv[i][e];
        }
      if (AHEAD) fetch(next);
      next = offset(j + (AHEAD ? 2 : 1) * GROUPS);
#pragma unroll
      for (int r = 0; r < PS_ROWS; ++r) {
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
        x = (x - slope[r] * float(last - j)) * kLog2e;
        if (!seen) continue;
        if (x > m[r]) {
          const float f = ex2(m[r] - x);  // m = -infinity: 0
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
    // join the groups of a warp by exchange, the warps in shared memory
#pragma unroll
    for (int r = 0; r < PS_ROWS; ++r) {
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
    const bool all = at.t == 0 && n == at.v.units;
    float* slot = d.slots + (int64_t(blockIdx.x) + int64_t(at.b) * d.segs + at.s) * d.rows * LD;
    for (int i = threadIdx.x; i < rows * D; i += PD_THREADS) {
      const int r = i / D, e = i - r * D;
      float mm = -INFINITY;
#pragma unroll
      for (int w = 0; w < PD_THREADS / 32; ++w) mm = fmaxf(mm, acc[w][r][32 * NI]);
      const float z = mm == -INFINITY ? 0.f : mm;
      float x = 0.f, sum = 0.f;
#pragma unroll
      for (int w = 0; w < PD_THREADS / 32; ++w) {
        const float f = ex2(acc[w][r][32 * NI] - z);
        x += f * acc[w][r][e];
        sum += f * acc[w][r][32 * NI + 1];
      }
      if (all) {
        store_elem(a.out, a.dtype, at.b * a.o_stride_t + (first + r) * a.o_stride_h + e, sum == 0.f ? 0.f : x / sum);
        if (a.lse && e == 0) a.lse[int64_t(at.b) * a.n_q_heads + first + r] = (mm + log2f(sum)) * kLn2;
      } else {
        slot[r * LD + e] = x;
        if (e == 0) {
          slot[r * LD + D] = mm;
          slot[r * LD + D + 1] = sum;
        }
      }
    }
    left -= n;
    if (left > 0) {
      at.t += n - 1;
      at.next(d);
    }
  }
}

// ---------------------------------------------------------------- join
// One CTA a (request, query head): the slots of its segment in CTA order.
__global__ void __launch_bounds__(PD_THREADS) paged_join_kernel(const __grid_constant__ DecodeParamsX d, int tile_rows) {
  __shared__ int64_t warp_sums[PD_THREADS / 32];
  __shared__ int64_t my_first;
  __shared__ float reduce[PD_THREADS / 32];
  extern __shared__ float slots_of[];  // [2][grid]
  float *factor = slots_of, *part = slots_of + d.grid;
  const PagedParams& p = d.p;
  const smaq_paged_args& a = p.a;
  const int b = blockIdx.x / a.n_q_heads, h = blockIdx.x - b * a.n_q_heads, D = a.head_dim, LD = D + 2;
  const int kvh = h / p.group, tile = (h - kvh * p.group) / tile_rows, r = h - kvh * p.group - tile * tile_rows;
  const int s = kvh * d.tiles + tile;
  int64_t costs = 0;
  for (int b0 = 0; b0 < a.batch; b0 += PD_THREADS) {
    int64_t before;
    const int64_t chunk = block_prefix(packed_cost(d, b0 + threadIdx.x), warp_sums, before);
    if (b0 + int(threadIdx.x) == b) my_first = (costs + before) >> PD_PACK;
    costs += chunk;
  }
  __syncthreads();
  const int64_t total = costs >> PD_PACK;
  const int units = visible(p, b).units;
  pdl_wait();  // the slots are complete from here on; every CTA waits, so this grid ends after the other
  if (units == 0) return;
  const int64_t f = my_first + int64_t(s) * (units + PD_START) + PD_START, e = f + units - 1;
  const int c0 = run_of(f, total, d.grid), c1 = run_of(e, total, d.grid);
  if (c0 == c1) return;
  const int64_t step = int64_t(d.rows) * LD;
  const float* slot = d.slots + (int64_t(c0) + int64_t(b) * d.segs + s) * step + r * LD;
  const int n = c1 - c0 + 1;  // at most the grid
  // every slot's maximum and sum at once, then its factor
  float m = -INFINITY;
  for (int i = threadIdx.x; i < n; i += PD_THREADS) {
    const float* ml = slot + i * step + D;  // two scalars: at odd head dims a slot's rows start at odd floats
    factor[i] = ml[0];
    part[i] = ml[1];
    m = fmaxf(m, factor[i]);
  }
  m = warp_max(m);
  if ((threadIdx.x & 31) == 0) reduce[threadIdx.x >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < PD_THREADS / 32; ++i) m = fmaxf(m, reduce[i]);
  const float z = m == -INFINITY ? 0.f : m;
  float sum = 0.f;
  for (int i = 0; i < n; ++i) sum += ex2(factor[i] - z) * part[i];  // in slot order, by every thread alike
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += PD_THREADS) factor[i] = ex2(factor[i] - z);
  __syncthreads();
  const float inv = sum == 0.f ? 0.f : 1.0f / sum;
  for (int c = threadIdx.x; c < D; c += PD_THREADS) {
    float x = 0.f;
#pragma unroll 8
    for (int i = 0; i < n; ++i) x += factor[i] * slot[i * step + c];
    store_elem(a.out, a.dtype, b * a.o_stride_t + h * a.o_stride_h + c, x * inv);
  }
  if (a.lse && threadIdx.x == 0) a.lse[int64_t(b) * a.n_q_heads + h] = (m + log2f(sum)) * kLn2;
}

constexpr int PS_CTAS = 4;  // CTAs an SM of the SIMT kernel

// Which kernel: the ring kernels take head_dim 64, 128 and (16-bit) 256 on 16-byte boundaries.
enum { PATH_SIMT, PATH_MMA, PATH_F32 };
struct Shape {
  int path, tile, ctas;  // query heads a tile, CTAs an SM
};
Shape shape_of(int dtype, int head_dim, int group, bool aligned) {
  const bool ring = aligned && (head_dim == 64 || head_dim == 128 || (head_dim == 256 && dtype != SMAQ_F32));
  if (!ring) return {PATH_SIMT, PS_ROWS, PS_CTAS};
  if (dtype == SMAQ_F32) return {PATH_F32, group > 4 ? 8 : 4, head_dim == 64 ? 2 : 1};
  return {PATH_MMA, 16, head_dim == 256 ? 1 : 2};
}

template <class K>
int launch_ring(K kern, int smem, const DecodeParamsX& d, cudaStream_t st) {
  if (const int rc = allow_smem(reinterpret_cast<const void*>(kern), smem, "paged_decode")) return rc;
  kern<<<d.grid, PD_THREADS, smem, st>>>(d);
  return cuda_status(cudaGetLastError(), "paged_decode");
}
template <class DT, int D>
int launch_mma(const DecodeParamsX& d, cudaStream_t st) {
  switch (cap_mode(d.p.a)) {
    case CAP_NONE: return launch_ring(paged_decode_kernel<DT, D, CAP_NONE>, Cfg<D>::SMEM, d, st);
    case CAP_LOW: return launch_ring(paged_decode_kernel<DT, D, CAP_LOW>, Cfg<D>::SMEM, d, st);
    default: return launch_ring(paged_decode_kernel<DT, D, CAP_ANY>, Cfg<D>::SMEM, d, st);
  }
}
template <class DT>
int launch_mma_dim(const DecodeParamsX& d, cudaStream_t st) {
  switch (d.p.a.head_dim) {
    case 64: return launch_mma<DT, 64>(d, st);
    case 128: return launch_mma<DT, 128>(d, st);
    default: return launch_mma<DT, 256>(d, st);
  }
}
template <int D, int R>
int launch_f32(const DecodeParamsX& d, cudaStream_t st) {
  return d.p.a.softcap > 0.f ? launch_ring(paged_decode_f32_kernel<D, R, true>, FCfg<D, R>::SMEM, d, st)
                             : launch_ring(paged_decode_f32_kernel<D, R, false>, FCfg<D, R>::SMEM, d, st);
}
template <class DT>
int launch_simt(const DecodeParamsX& d, cudaStream_t st) {
  const int D = d.p.a.head_dim;
  const bool vec = D % 4 == 0 && paged_aligned(d.p.a);
  auto go = [&](auto kern) {
    kern<<<d.grid, PD_THREADS, 0, st>>>(d);
    return cuda_status(cudaGetLastError(), "paged_decode");
  };
  if (D <= 64) return vec ? go(paged_simt_kernel<DT, 2, true>) : go(paged_simt_kernel<DT, 2, false>);
  if (D <= 128) return vec ? go(paged_simt_kernel<DT, 4, true>) : go(paged_simt_kernel<DT, 4, false>);
  return vec ? go(paged_simt_kernel<DT, 8, true>) : go(paged_simt_kernel<DT, 8, false>);
}

}  // namespace

}  // namespace smaq

extern "C" size_t smaq_paged_decode_workspace_size(int batch, int n_q_heads, int n_kv_heads, int head_dim) {
  using namespace smaq;
  if (batch <= 0 || n_kv_heads <= 0 || n_q_heads < n_kv_heads || head_dim <= 0) return 0;
  // enough for whichever kernel the dtype and alignment choose
  const int group = n_q_heads / n_kv_heads;
  size_t most = 0;
  for (const int dtype : {SMAQ_F32, SMAQ_BF16})
    for (const bool aligned : {false, true}) {
      const Shape s = shape_of(dtype, head_dim, group, aligned);
      const int tiles = (group + s.tile - 1) / s.tile, rows = group < s.tile ? group : s.tile;
      const size_t n = (size_t(num_sms()) * s.ctas + size_t(batch) * n_kv_heads * tiles) * rows * (head_dim + 2) * sizeof(float);
      most = n > most ? n : most;
    }
  return most;
}

extern "C" int smaq_paged_decode(const smaq_paged_args* args, void* stream) {
  using namespace smaq;
  DecodeParamsX d;
  if (const int st = paged_check(args, false, d.p)) return st;
  const smaq_paged_args& a = d.p.a;
  if (a.n_rows != a.batch) return fail(SMAQ_ERR_INVALID, "paged_decode: %lld rows for batch %d (one row a request)", (long long)a.n_rows, a.batch);
  if (a.batch == 0) return SMAQ_OK;
  if (a.batch >= 1 << PD_PACK) return fail(SMAQ_ERR_UNSUPPORTED, "paged_decode: batch %d", a.batch);
  const size_t need = smaq_paged_decode_workspace_size(a.batch, a.n_q_heads, a.n_kv_heads, a.head_dim);
  if (!a.workspace || a.workspace_bytes < need)
    return fail(SMAQ_ERR_WORKSPACE, "paged_decode: workspace %zu bytes, needs %zu", a.workspace ? a.workspace_bytes : size_t(0), need);
  if (reinterpret_cast<uintptr_t>(a.workspace) % 16) return fail(SMAQ_ERR_INVALID, "paged_decode: workspace must be 16-byte aligned");
  const Shape sh = shape_of(a.dtype, a.head_dim, d.p.group, paged_aligned(a));
  d.tiles = (d.p.group + sh.tile - 1) / sh.tile;
  d.rows = d.p.group < sh.tile ? d.p.group : sh.tile;
  d.segs = a.n_kv_heads * d.tiles;
  d.grid = num_sms() * sh.ctas;
  d.slots = static_cast<float*>(a.workspace);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  int rc;
  if (sh.path == PATH_MMA) rc = a.dtype == SMAQ_BF16 ? launch_mma_dim<BF16>(d, st) : launch_mma_dim<F16>(d, st);
  else if (sh.path == PATH_F32)
    rc = a.head_dim == 64 ? (sh.tile == 4 ? launch_f32<64, 4>(d, st) : launch_f32<64, 8>(d, st))
                          : (sh.tile == 4 ? launch_f32<128, 4>(d, st) : launch_f32<128, 8>(d, st));
  else rc = a.dtype == SMAQ_F32 ? launch_simt<F32>(d, st) : a.dtype == SMAQ_BF16 ? launch_simt<BF16>(d, st) : launch_simt<F16>(d, st);
  if (rc) return rc;
  // tables or windows of one unit: no segment can have been split
  if (int64_t(a.max_blocks) * a.page_size <= PD_UNIT || (a.window > 0 && a.window <= PD_UNIT)) return SMAQ_OK;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(a.batch) * unsigned(a.n_q_heads));
  cfg.blockDim = dim3(PD_THREADS);
  cfg.dynamicSmemBytes = size_t(d.grid) * 2 * sizeof(float);
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, paged_join_kernel, d, sh.tile), "paged_decode join");
}
