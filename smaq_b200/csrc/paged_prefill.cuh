// Tiles, visibility and the exact row of the prefill kernels.
#pragma once
#include "paged.cuh"

namespace smaq {

// The rows of a request and KV head are its tokens times the group's query heads: row f is token f / group,
// head f % group.  A tile is `rows` consecutive ones.
struct PrefillTile {
  int b;         // request
  int f0;        // first row
  int rows;      // rows of the request from f0 on, up to the tile's size; 0: no tile
  int first;     // row in q of the request's first token
  int past;      // position of the request's first token: seq_len - tokens (may be negative)
  int len;       // seq_len
  int prefix;    // tokens that every row sees
  int lo, hi;    // tokens that the tile's rows see lie in [0, prefix) or [lo, hi)
};

__device__ __forceinline__ int cu_at(const PagedParams& p, int b) {
  return int(min(int64_t(max(__ldg(p.a.cu_query + b), 0)), p.a.n_rows));
}

// Tile `x` (counted over all requests) for blocks of THREADS threads, as long as the tiles of `size` rows reach
// (rows 0: no such tile).  Every thread loads one request's facts at once, and the one whose request it is fills `out`.
// `sums` and `out` are shared; all threads return the same.
template <int THREADS>
__device__ __forceinline__ PrefillTile find_tile(const PagedParams& p, int x, int size, bool reverse, int* sums, PrefillTile* out) {
  const int B = p.a.batch, lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  int total = 0, mine = 0, before = 0, c0 = 0, c1 = 0, len = 0, prefix = 0;
  auto step = [&](int b0) {
    const int b = b0 + threadIdx.x;
    mine = 0;
    if (b < B) {
      c0 = cu_at(p, b);
      c1 = cu_at(p, b + 1);
      len = paged_len(p, b);
      prefix = p.a.prefix_lens ? min(max(__ldg(p.a.prefix_lens + b), 0), len) : 0;
      mine = int((int64_t(max(c1 - c0, 0)) * p.group + size - 1) / size);
    }
    int v = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(~0u, v, o);
      if (lane >= o) v += u;
    }
    __syncthreads();
    if (lane == 31) sums[w] = v;
    __syncthreads();
    int all = 0, base = 0;
#pragma unroll
    for (int i = 0; i < THREADS / 32; ++i) {
      if (i < w) base += sums[i];
      all += sums[i];
    }
    before = base + v - mine;
    return all;
  };
  if (threadIdx.x == 0) out->rows = 0;
  for (int b0 = 0; b0 < B; b0 += THREADS) total += step(b0);
  if (x < total) {
    if (reverse) x = total - 1 - x;
    int base = 0;
    for (int b0 = 0; b0 < B && base <= x; b0 += THREADS) {
      const int all = B <= THREADS ? total : step(b0);
      if (x >= base + before && x < base + before + mine) {
        PrefillTile t;
        const int n = c1 - c0;
        t.b = b0 + threadIdx.x;
        t.f0 = (x - base - before) * size;
        t.first = c0;
        t.len = len;
        t.past = len - n;
        t.prefix = prefix;
        t.rows = int(min(int64_t(size), int64_t(n) * p.group - t.f0));
        const int i0 = t.past + t.f0 / p.group, i1 = t.past + (t.f0 + t.rows - 1) / p.group;
        t.hi = max(min(i1 + 1, t.len), 0);
        t.lo = p.a.window > 0 ? min(max(i0 - p.a.window + 1, 0), t.hi) : 0;
        *out = t;
      }
      base += all;
    }
  }
  __syncthreads();
  return *out;
}

// Tiles of `size` rows that any cu_query of this many rows and requests can have: sum of ceil(x_b / size).
inline int64_t most_tiles(int64_t n_rows, int batch, int group, int size) {
  return (n_rows * group + int64_t(batch) * (size - 1)) / size;
}

// Whether some row of the tile sees token j: others are read as zeros.
__device__ __forceinline__ bool tile_sees(const PrefillTile& t, int j) { return j < t.prefix || (j >= t.lo && j < t.hi); }
// Whether the row of position i sees token j < len.
__device__ __forceinline__ bool row_sees(const PagedParams& p, const PrefillTile& t, int i, int j) {
  return j < t.prefix || (j <= i && (p.a.window == 0 || j > i - p.a.window));
}

// Blocks of N tokens that a tile walks: those of the prefix, then those of [lo, hi).
struct PrefillBlocks {
  int head, jump, count;
  PrefillBlocks() = default;
  __device__ __forceinline__ PrefillBlocks(const PrefillTile& t, int N) {
    head = (t.prefix + N - 1) / N;
    const int from = max(head, t.lo / N), to = (t.hi + N - 1) / N;
    jump = from - head;
    count = head + max(to - from, 0);
  }
  __device__ __forceinline__ int base(int k, int N) const { return (k < head ? k : k + jump) * N; }
};

// Rows before the first request's and past the last one's: zeros for this block's share.
__device__ __forceinline__ void write_padding(const PagedParams& p, int kvh, int block, int blocks) {
  const smaq_paged_args& a = p.a;
  const int64_t end = a.batch ? cu_at(p, a.batch) : 0, head = a.batch ? min(int64_t(cu_at(p, 0)), end) : 0;
  for (int64_t r = block; r < head + a.n_rows - end; r += blocks) {
    const int64_t t = r < head ? r : r - head + end;
    for (int i = threadIdx.x; i < p.group * a.head_dim; i += blockDim.x) {
      const int h = kvh * p.group + i / a.head_dim;
      store_elem(a.out, a.dtype, t * a.o_stride_t + h * a.o_stride_h + i % a.head_dim, 0.f);
      if (a.lse && i % a.head_dim == 0) a.lse[t * a.n_q_heads + h] = -INFINITY;
    }
  }
}

// Whether one of eight 16-bit elements is an infinity or NaN.
template <class DT>
__device__ __forceinline__ bool any_special(uint4 v) {
  constexpr uint32_t E = DT::code == SMAQ_F16 ? 0x7C007C00u : 0x7F807F80u;
  auto one = [](uint32_t w) { return (w & E & 0xFFFFu) == (E & 0xFFFFu) || (w & E >> 16 << 16) == (E >> 16 << 16); };
  return one(v.x) || one(v.y) || one(v.z) || one(v.w);
}

// One row by one warp over its visible tokens alone, in 32 bits.  The matrix kernels multiply the values of
// tokens that a row does not see by a weight of zero, which an infinity or NaN there turns into NaN.  They
// look for such values in the blocks that some rows see in part, and only where there is one are that
// tile's rows without a finite result redone here.  That is slow: 8192 tokens at 32/8 heads, one infinity
// at token 3203, whose tile has 256 rows to redo: 239 ms instead of 0.6.
static __device__ __noinline__ void exact_row(const PagedParams& p, const PrefillTile& t, int kvh, int f) {
  const smaq_paged_args& a = p.a;
  const int lane = threadIdx.x & 31, D = a.head_dim;
  const int tok = f / p.group, h = kvh * p.group + f % p.group, i = t.past + tok;
  const int64_t qo = int64_t(t.first + tok) * a.q_stride_t + h * a.q_stride_h;
  const int32_t* table = a.block_table + t.b * a.table_stride;
  const float slope = a.slopes ? a.slopes[h] : 0.f;
  float m = -INFINITY, s = 0.f, o[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) o[k] = 0.f;
  for (int j = 0; j < max(t.prefix, t.hi); ++j) {
    if (!row_sees(p, t, i, j)) continue;
    const int64_t off = token_offset(p, table, j) + kvh * a.c_stride_h;
    float x = 0.f;
    for (int e = lane; e < D; e += 32) x = fmaf(load_elem(a.q, a.dtype, qo + e), load_elem(a.k_cache, a.dtype, off + e), x);
    x = warp_sum(x) * a.scale;
    if (a.softcap > 0.f) x = a.softcap * tanhf(x / a.softcap);
    x = (x - slope * fabsf(float(i - j))) * kLog2e;
    const float n = x > m ? x : m, f1 = m == -INFINITY ? 0.f : ex2(m - n), w = ex2(x - (n == -INFINITY ? 0.f : n));
    m = n;
    s = s * f1 + w;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int e = lane + 32 * k;
      if (e < D) o[k] = o[k] * f1 + w * load_elem(a.v_cache, a.dtype, off + e);
    }
  }
  const int64_t oo = int64_t(t.first + tok) * a.o_stride_t + h * a.o_stride_h;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const int e = lane + 32 * k;
    if (e < D) store_elem(a.out, a.dtype, oo + e, s == 0.f ? 0.f : o[k] / s);
  }
  if (a.lse && lane == 0) a.lse[int64_t(t.first + tok) * a.n_q_heads + h] = (m + log2f(s)) * kLn2;
}

}  // namespace smaq
