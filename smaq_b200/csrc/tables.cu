// Block tables and slot maps of one serving step, built on the GPU from request lengths.
//
// With s tokens a page, request b holds h_b = ceil(c_b / s) pages and needs
// d_b = ceil((c_b + n_b) / s) - h_b more.  R = the finished requests' pages, T = F + sum R is the
// stack's height after they are pushed, P_b = d_0 + .. + d_b: b is admitted when d_b = 0 or P_b <= T,
// and its i-th new page is stack entry T - 1 - (P_b - d_b) - i.  An entry at or above F is read from
// the finished request's own table row, so nothing read here is written here and one launch does it.
//
// Every CTA redoes the three prefix sums (batch is small: two steps of 512 for 1001 requests) and
// then serves its share of the tokens, four consecutive ones a thread: the request is found by
// bisection in shared memory once, and a page is looked up once per page.  The token that opens a page
// writes the table entry.  Bound by latency (lengths -> sums -> stack -> stores), not by bytes.
// On the device 64 requests of one token take 8.2 us, 1001 requests with 285K tokens 11.4 us (0.6 us of bytes).
#include "common.cuh"

namespace smaq {

namespace {

constexpr int TB_THREADS = 512;
constexpr int TB_PER = 4;            // tokens a thread
constexpr int TB_MAX_BATCH = 16384;  // 12 bytes of shared memory a request

constexpr int kMost = 0x7FFFFFFF;

// Sums of non-negative numbers, at most 2^31 - 1: lengths come from the device and may be anything.
__device__ __forceinline__ int add(int a, int b) { return int(min(unsigned(a) + unsigned(b), unsigned(kMost))); }
__device__ __forceinline__ int3 add3(int3 a, int3 b) { return make_int3(add(a.x, b.x), add(a.y, b.y), add(a.z, b.z)); }
__device__ __forceinline__ int pages_of(int tokens, int s) { return int((unsigned(tokens) + unsigned(s) - 1u) / unsigned(s)); }

// Inclusive prefix sum over the block of one int3 a thread; `total` gets the block's sum.
__device__ __forceinline__ int3 scan3(int3 v, int3* warp_sums, int3& total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int3 u = make_int3(__shfl_up_sync(~0u, v.x, o), __shfl_up_sync(~0u, v.y, o), __shfl_up_sync(~0u, v.z, o));
    if (lane >= o) v = add3(v, u);
  }
  if (lane == 31) warp_sums[w] = v;
  __syncthreads();
  int3 before = make_int3(0, 0, 0);
  total = before;
  for (int i = 0; i < TB_THREADS / 32; ++i) {
    if (i < w) before = add3(before, warp_sums[i]);
    total = add3(total, warp_sums[i]);
  }
  __syncthreads();
  return add3(v, before);
}

// Smallest b with x < a[b] for ascending a[0 .. n).
__device__ __forceinline__ int first_above(const int* a, int n, int x) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (x < a[mid]) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

__global__ void __launch_bounds__(TB_THREADS) step_tables_kernel(const __grid_constant__ smaq_tables_args a) {
  extern __shared__ int smem[];
  int* upto = smem;             // [B] tokens up to and with request b
  int* base = smem + a.batch;   // [B] page j of request b (j >= h_b) is stack entry base - j; < 0: not admitted
  int* back = base + a.batch;   // [B] pages given back up to and with request b
  __shared__ int3 warp_sums[TB_THREADS / 32];
  __shared__ int used, opened;  // pages taken; tokens up to the last request that took one
  const int B = a.batch, s = a.page_size, M = a.max_blocks;
  const int F = min(max(*a.free_count, 0), int(a.pool_size));
  const int room = int(min(int64_t(M) * s, int64_t(kMost) - 1));  // tokens that a table row holds
  if (threadIdx.x == 0) used = opened = 0;
  int3 carry = make_int3(0, 0, 0);
  for (int b0 = 0; b0 < B; b0 += TB_THREADS) {
    const int b = b0 + threadIdx.x;
    int3 v = make_int3(0, 0, 0);
    if (b < B) {
      const int c = max(a.context_lens[b], 0), n = max(a.query_lens[b], 0), held = pages_of(c, s);
      if (a.finished && a.finished[b]) {
        v.z = min(held, M);
      } else {
        v.x = n;
        v.y = n > 0 && add(c, n) <= room ? pages_of(c + n, s) - held : 0;
      }
    }
    int3 total;
    v = add3(scan3(v, warp_sums, total), carry);
    carry = add3(carry, total);
    if (b < B) {
      upto[b] = v.x;
      base[b] = v.y;
      back[b] = v.z;
    }
  }
  __syncthreads();
  const int top = add(F, carry.z);
  for (int b = threadIdx.x; b < B; b += TB_THREADS) {
    const int c = max(a.context_lens[b], 0), n = upto[b] - (b ? upto[b - 1] : 0);
    const int held = pages_of(c, s), total = base[b];
    const bool over = a.finished && a.finished[b], fits = !over && add(c, n) <= room && upto[b] < kMost;
    const int need = fits && n > 0 ? pages_of(c + n, s) - held : 0;
    const bool ok = fits && (need == 0 || total <= top);
    // written over what only this thread reads
    base[b] = ok ? add(max(top - 1 - (total - need), 0), held) : -1;
    if (ok && need) {
      atomicMax(&used, total);
      atomicMax(&opened, upto[b]);
    }
    if (blockIdx.x == 0) {
      a.cu_query[b + 1] = upto[b];
      a.seq_lens[b] = ok ? c + n : 0;
      a.admitted[b] = ok;
    }
  }
  __syncthreads();
  const int left = top - used;
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    a.cu_query[0] = 0;
    *a.free_count_out = left;
  }
  // stack entry p at or above F: the finished requests' pages, in order
  auto given = [&](int p) {
    const int r = min(first_above(back, B, p - F), B - 1);
    return a.block_table[r * a.table_stride + (p - F - (r ? back[r - 1] : 0))];
  };
  const int64_t tid = int64_t(blockIdx.x) * TB_THREADS + threadIdx.x, threads = int64_t(gridDim.x) * TB_THREADS;
  for (int64_t p = F + tid; p < left && p < a.pool_size; p += threads) a.free_blocks[p] = given(int(p));

  const int tokens = B ? upto[B - 1] : 0;
  // tokens past n_tokens have no slot to report, but the pages they open are the request's all the same
  const int64_t end = max(a.n_tokens, int64_t(opened));
  for (int64_t t0 = tid * TB_PER; t0 < end; t0 += threads * TB_PER) {
    int pos[TB_PER];
    int64_t slot[TB_PER];
    int b = -1, next = 0, page = 0, blk = -1, off = 0, p = 0;
#pragma unroll
    for (int i = 0; i < TB_PER; ++i) {
      const int64_t t = t0 + i;
      pos[i] = 0;
      slot[i] = -1;
      if (t >= tokens) continue;
      if (b < 0 || t >= next) {  // a request begins
        b = first_above(upto, B, int(t));
        next = upto[b];
        p = max(a.context_lens[b], 0) + int(t) - (b ? upto[b - 1] : 0);
        blk = p / s;
        off = p - blk * s;
        page = -1;
      } else {
        ++p;
        if (++off == s) {
          off = 0;
          ++blk;
          page = -1;
        }
      }
      pos[i] = p;
      if (base[b] < 0) continue;
      if (page < 0) {
        const int held = pages_of(max(a.context_lens[b], 0), s);
        if (blk < held) {
          page = a.block_table[b * a.table_stride + blk];
        } else {
          const int e = base[b] - blk;
          page = e < F ? a.free_blocks[e] : given(e);
          if (off == 0) a.block_table[b * a.table_stride + blk] = page;
        }
      }
      slot[i] = int64_t(page) * s + off;
    }
    if (t0 + TB_PER <= a.n_tokens) {  // buffers are 16-byte aligned, t0 a multiple of 4
      *reinterpret_cast<int4*>(a.positions + t0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
      *reinterpret_cast<longlong2*>(a.slots + t0) = make_longlong2(slot[0], slot[1]);
      *reinterpret_cast<longlong2*>(a.slots + t0 + 2) = make_longlong2(slot[2], slot[3]);
    } else {
      for (int i = 0; i < TB_PER && t0 + i < a.n_tokens; ++i) {
        a.positions[t0 + i] = pos[i];
        a.slots[t0 + i] = slot[i];
      }
    }
  }
}

}  // namespace

}  // namespace smaq

extern "C" int smaq_step_tables(const smaq_tables_args* args, void* stream) {
  using namespace smaq;
  if (!args) return fail(SMAQ_ERR_INVALID, "step_tables: null arguments");
  const smaq_tables_args& a = *args;
  if (a.batch < 0 || a.n_tokens < 0 || a.pool_size < 0 || a.pool_size >= (int64_t(1) << 31) || a.max_blocks < 0 || a.page_size < 1)
    return fail(SMAQ_ERR_INVALID, "step_tables: bad sizes (batch %d, tokens %lld, page_size %d)", a.batch,
                (long long)a.n_tokens, a.page_size);
  if (a.batch > TB_MAX_BATCH) return fail(SMAQ_ERR_UNSUPPORTED, "step_tables: batch %d above %d", a.batch, TB_MAX_BATCH);
  if (a.n_tokens >= (int64_t(1) << 31)) return fail(SMAQ_ERR_UNSUPPORTED, "step_tables: 2^31 tokens or more");
  if (!a.free_count || !a.free_count_out || !a.cu_query || (a.pool_size && !a.free_blocks) ||
      (a.batch && (!a.context_lens || !a.query_lens || !a.seq_lens || !a.admitted || (a.max_blocks && !a.block_table))) ||
      (a.n_tokens && (!a.positions || !a.slots)))
    return fail(SMAQ_ERR_INVALID, "step_tables: null pointer");
  if (a.table_stride < a.max_blocks) return fail(SMAQ_ERR_INVALID, "step_tables: table stride below its width");
  if (reinterpret_cast<uintptr_t>(a.positions) % 16 || reinterpret_cast<uintptr_t>(a.slots) % 16)
    return fail(SMAQ_ERR_INVALID, "step_tables: positions and slots must be 16-byte aligned");
  const size_t bytes = size_t(a.batch) * 12;
  if (bytes > 40 * 1024)  // 48 KB without a grant, the static variables included
    if (const int rc = allow_smem(reinterpret_cast<const void*>(step_tables_kernel), TB_MAX_BATCH * 12, "step_tables")) return rc;
  const int64_t want = (a.n_tokens + TB_THREADS * TB_PER - 1) / (TB_THREADS * TB_PER);
  const int grid = int(want < 1 ? 1 : want < num_sms() ? want : num_sms());
  step_tables_kernel<<<grid, TB_THREADS, bytes, static_cast<cudaStream_t>(stream)>>>(a);
  return cuda_status(cudaGetLastError(), "step_tables");
}
