// Prefill attention on the 5th-generation tensor cores (bf16 / fp16, head_dim 64 and 128).
//
// A CTA holds 256 rows (tokens times grouped heads, paged_prefill.cuh) as two tiles of 128 and walks blocks of 128
// tokens.  For each tile and block S = Q K^T goes to tensor memory, a warpgroup turns it into weights P there, and
// O += P V reads P from tensor memory.  The two tiles take turns: while one is in its softmax the tensor cores work for
// the other.
//   warps 0-3, 4-7   softmax of tile 0, 1: thread = row, so maximum and sum need no exchange;
//   warps 8-11       copies: queries once, then keys and values (cp.async of 16 bytes through the block table, written in the
//                    128-byte swizzled operand layout; tokens that no row sees are written as zeros);
//   warp 12          one thread issues all products (warps 13-15 only lend their registers).
// Tensor memory: S0 S1 (128 columns each), O0 O1 (head_dim each); P overwrites its S.  The product for the next S of a tile is
// issued right behind the product that reads its P, and its completion also says that O is at rest: a softmax warp may
// then rescale O, which it does only when a row's maximum grew by more than 2^8 (the reference maximum of a row
// lags by at most that, so weights stay below 2^8 in either type).
// Weights are rounded once, to the cache's type; the sums are of the unrounded ones.
// Every wait is bounded; one that runs out sets g_prefill_fault and the CTA drains.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <mutex>

#include "paged_prefill.cuh"
#include "prefill_tc.cuh"
#include "tcgen05.cuh"

namespace smaq {

namespace {

using namespace tc5;

__device__ unsigned int g_prefill_fault;

constexpr int PT_THREADS = 512;
constexpr int PT_N = 128;                 // tokens a block
constexpr int PT_ROWS = 256;
constexpr int PT_LOAD_WARP = 8, PT_MMA_WARP = 12;
constexpr uint32_t PT_COLS = 512;
constexpr float PT_LAG = 8.0f;            // log2
constexpr uint32_t PT_SPIN = 1u << 24;    // polls before a wait gives up

// The whole warp waits, and gives up together.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity) { return __all_sync(~0u, mbar_wait(bar, parity, PT_SPIN)); }

template <int D>
struct PtCfg {
  static constexpr int TILE = 128 * D * 2;              // bytes: 128 rows of queries, keys or values
  static constexpr int STAGES = 2;
  static constexpr int SMEM = 2 * TILE + 2 * STAGES * TILE + 1024;
};

struct PtParams {
  PagedParams p;
  int tma;         // keys and values come through the tensor maps where every token of a block is seen
  int box;         // slots a box: page_size, at most PT_N
  CUtensorMap k, v;
};

struct PtBars {
  uint64_t q_full, k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_ready[2], o_full[2];
  uint32_t tmem;
  int special;
};

template <class DT, int D, bool MOD>
__global__ void __launch_bounds__(PT_THREADS, 1) prefill_tc_kernel(const __grid_constant__ PtParams pt) {
  using T = typename DT::T;
  const PagedParams& p = pt.p;
  constexpr int TILE = PtCfg<D>::TILE, STAGES = PtCfg<D>::STAGES, CH = D / 8, ATOM = 128 * 128;
  constexpr uint32_t ID_S = idesc(DT::code == SMAQ_BF16, PT_N, false), ID_O = idesc(DT::code == SMAQ_BF16, D, true);
  extern __shared__ uint8_t smem_raw[];
  __shared__ PtBars bars;
  __shared__ int sums[PT_THREADS / 32], found[2];
  const smaq_paged_args& a = p.a;
  const uint32_t base_raw = smem_u32(smem_raw), pad = (1024u - (base_raw & 1023u)) & 1023u;
  uint8_t* smem = smem_raw + pad;
  const uint32_t qs = base_raw + pad, ks = qs + 2 * TILE, vs = ks + STAGES * TILE;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, kvh = int(blockIdx.x % unsigned(a.n_kv_heads)), tile = int(blockIdx.x / unsigned(a.n_kv_heads));

  write_padding(p, kvh, tile, int(gridDim.x / unsigned(a.n_kv_heads)));
  const PrefillTile t = find_tile<PT_THREADS>(p, tile, PT_ROWS, true, sums, found);
  if (t.rows == 0) return;
  const PrefillBlocks blocks(t, PT_N);
  const int n = blocks.count, tiles = t.rows > 128 ? 2 : 1;

  if (threadIdx.x == 0) {
    mbar_init(&bars.q_full, 128);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&bars.k_full[s], 128);
      mbar_init(&bars.v_full[s], 128);
      mbar_init(&bars.k_empty[s], 1);
      mbar_init(&bars.v_empty[s], 1);
      mbar_init(&bars.s_full[s], 1);
      mbar_init(&bars.p_ready[s], 128);
      mbar_init(&bars.o_full[s], 1);
    }
    bars.special = 0;
    fence_mbar_init();
  }
  if (warp == PT_MMA_WARP) alloc(&bars.tmem, PT_COLS);
  fence_before();
  __syncthreads();
  fence_after();
  constexpr uint32_t tmem = 0;  // all 512 columns are this CTA's: the allocation starts at 0
  const uint32_t s_col = 0, o_col = 256;  // S of tile i at s_col + 128 i, O at o_col + D i
  bool failed = false;

  const int last = t.f0 + t.rows;
  const int least = t.past + fast_div(t.f0, p.group_div), most = t.past + fast_div(last - 1, p.group_div);
  auto seen_by_all = [&](int base) {
    return base + PT_N <= t.prefix || (base + PT_N <= least + 1 && (a.window == 0 || base > most - a.window));
  };
  float odd = 0.f, l = 0.f;  // softmax threads: NaN where an output is not finite; sum of weights
  int f = 0;

  if (warp >= PT_LOAD_WARP) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp < PT_MMA_WARP) {
      // ---- copies: warp w brings rows 32w .. 32w + 31 of every operand
      const int w = warp - PT_LOAD_WARP, tid = threadIdx.x - PT_LOAD_WARP * 32;
      for (int i = tid; i < tiles * 128 * CH; i += 128) {
        const int r = i / CH, ch = i % CH, fr = t.f0 + r, tok = fast_div(fr, p.group_div);
        const bool live = r < t.rows;
        const T* src = static_cast<const T*>(a.q) + (live ? (t.first + tok) * a.q_stride_t + (kvh * p.group + fr - tok * p.group) * a.q_stride_h + ch * 8 : 0);
        cp_async16(qs + uint32_t((r >> 7) * TILE + (ch >> 3) * ATOM + (r & 127) * 128 + (((ch & 7) ^ (r & 7)) << 4)), src, live ? 16u : 0u);
      }
      cp_async_commit();
      const int32_t* table = a.block_table + t.b * a.table_stride;
      auto look_up = [&](int k) {
        if (k >= n) return int64_t(-1);
        const int j = blocks.base(k, PT_N) + 32 * w + lane;
        return tile_sees(t, j) ? token_offset(p, table, j) + kvh * a.c_stride_h : int64_t(-1);
      };
      auto bring = [&](const void* cache, uint32_t dst, int64_t off) {
        constexpr int PER = 32 / CH;  // rows a pass
#pragma unroll
        for (int i = 0; i < 32 / PER; ++i) {
          const int rr = i * PER + lane / CH, ch = lane % CH, r = 32 * w + rr;
          const int64_t o = __shfl_sync(~0u, off, rr);
          cp_async16(dst + uint32_t((ch >> 3) * ATOM + r * 128 + (((ch & 7) ^ (r & 7)) << 4)),
                     static_cast<const T*>(cache) + (o < 0 ? 0 : o) + ch * 8, o < 0 ? 0u : 16u);
        }
        cp_async_commit();
      };
      // copy g = 2 j brings keys of block j, 2 j + 1 its values; a copy is announced two copies later
      // values of a block that some rows see in part: look for infinities and NaN where this thread copies
      auto look_for_special = [&](int s) {
        bool odd_value = false;
        constexpr int PER = 32 / CH;
        for (int i = 0; i < 32 / PER; ++i) {
          const int ch = lane % CH, r = 32 * w + i * PER + lane / CH;
          odd_value |= any_special<DT>(*reinterpret_cast<const uint4*>(smem + (vs - qs) + s * TILE + (ch >> 3) * ATOM + r * 128 + (((ch & 7) ^ (r & 7)) << 4)));
        }
        if (odd_value) bars.special = 1;
      };
      auto announce = [&](int g) {
        const int j = g >> 1, s = j % STAGES;
        if ((g & 1) && !seen_by_all(blocks.base(j, PT_N))) look_for_special(s);
        fence_proxy_async_smem();
        mbar_arrive((g & 1) ? &bars.v_full[s] : &bars.k_full[s]);
      };
      if (pt.tma) {
        // A block whose every token is seen by some row comes in boxes of one page (or 128 slots of it) by 64
        // channels, a lane of warp 0 each; the others as below, announced at once.
        const int per = PT_N / pt.box, boxes = per * (D / 64);
        auto whole = [&](int k) {
          const int b = blocks.base(k, PT_N);
          return b + PT_N <= t.prefix || (b >= t.lo && b + PT_N <= t.hi);
        };
        auto page_of = [&](int k) {
          if (k >= n || lane >= boxes || !whole(k)) return 0;
          const int64_t blk = fast_div(blocks.base(k, PT_N) + (lane % per) * pt.box, p.page_div);
          return int(min(max(int64_t(__ldg(table + blk)), int64_t(0)), a.n_pages - 1));
        };
        auto fetch = [&](int j, int s, bool values, int page, int64_t off) {
          uint64_t* bar = values ? &bars.v_full[s] : &bars.k_full[s];
          const uint32_t dst = (values ? vs : ks) + s * TILE;
          if (whole(j)) {
            if (w == 0) {
              if (lane == 0) mbar_arrive_expect_tx(bar, TILE);
              __syncwarp();
              if (lane < boxes) {
                const int half = lane / per, b = lane % per, slot = blocks.base(j, PT_N) + b * pt.box;
                tma_4d(dst + half * ATOM + b * pt.box * 128, values ? &pt.v : &pt.k, half * 64, kvh, slot - fast_div(slot, p.page_div) * a.page_size, page, bar);
              }
              if (lane != 0) mbar_arrive(bar);
            } else {
              mbar_arrive(bar);
            }
            if (values && !seen_by_all(blocks.base(j, PT_N))) {
              if (!warp_wait(bar, (j / STAGES) & 1)) failed = true;
              look_for_special(s);
              fence_proxy_async_smem();  // before the stage is filled again
            }
            return;
          }
          bring(values ? a.v_cache : a.k_cache, dst, off);
          cp_async_wait<0>();
          announce(2 * j + values);
        };
        cp_async_wait<0>();
        fence_proxy_async_smem();
        mbar_arrive(&bars.q_full);
        int page = page_of(0);
        for (int j = 0; j < n; ++j) {
          const int s = j % STAGES;
          const uint32_t ph = uint32_t((j / STAGES) & 1) ^ 1u;
          const int next = page_of(j + 1);
          const int64_t off = whole(j) ? 0 : look_up(j);
          if (!warp_wait(&bars.k_empty[s], ph)) { failed = true; break; }
          fetch(j, s, false, page, off);
          if (!warp_wait(&bars.v_empty[s], ph)) { failed = true; break; }
          fetch(j, s, true, page, off);
          if (failed) break;
          page = next;
        }
      }
      int64_t off = pt.tma ? -1 : look_up(0);
      for (int j = 0; j < n && !failed && !pt.tma; ++j) {
        const int s = j % STAGES;
        const uint32_t ph = uint32_t((j / STAGES) & 1) ^ 1u;
        const int64_t next = look_up(j + 1);
        if (!warp_wait(&bars.k_empty[s], ph)) { failed = true; break; }
        bring(a.k_cache, ks + s * TILE, off);
        cp_async_wait<2>();
        if (j > 0) announce(2 * j - 2);
        if (!warp_wait(&bars.v_empty[s], ph)) { failed = true; break; }
        bring(a.v_cache, vs + s * TILE, off);
        cp_async_wait<2>();
        if (j == 0) {  // the queries were the group before the first keys
          fence_proxy_async_smem();
          mbar_arrive(&bars.q_full);
        } else {
          announce(2 * j - 1);
        }
        off = next;
      }
      cp_async_wait<0>();
      if (!failed && n > 0 && !pt.tma) {
        announce(2 * n - 2);
        announce(2 * n - 1);
      }
    } else if (warp == PT_MMA_WARP && n > 0) {
      // ---- products
      const uint32_t lead = elect_one();
      auto scores = [&](int i, int j) {
        const uint32_t q = qs + i * TILE, k = ks + (j % STAGES) * TILE;
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
          const uint32_t at = uint32_t((c >> 2) * ATOM + (c & 3) * 32);
          mma_ss(lead, tmem + s_col + 128 * i, desc(q + at, 16), desc(k + at, 16), ID_S, c > 0);
        }
        commit(lead, &bars.s_full[i]);
      };
      bool ok = warp_wait(&bars.q_full, 0) && warp_wait(&bars.k_full[0], 0);
      if (ok) {
        fence_after();
        for (int i = 0; i < tiles; ++i) scores(i, 0);
        commit(lead, &bars.k_empty[0]);
      }
      for (int j = 0; ok && j < n; ++j) {
        const int s = j % STAGES, s1 = (j + 1) % STAGES;
        ok = warp_wait(&bars.v_full[s], (j / STAGES) & 1);
        for (int i = 0; ok && i < tiles; ++i) {
          ok = warp_wait(&bars.p_ready[i], j & 1);
          if (!ok) break;
          fence_after();
#pragma unroll
          for (int c = 0; c < PT_N / 16; ++c)
            mma_ts(lead, tmem + o_col + D * i, tmem + s_col + 128 * i + 8 * c, desc(vs + s * TILE + c * 2048, ATOM), ID_O, (j > 0) | (c > 0));
          if (j + 1 < n) {
            if (i == 0) ok = warp_wait(&bars.k_full[s1], ((j + 1) / STAGES) & 1);
            if (!ok) break;
            fence_after();
            scores(i, j + 1);
          } else {
            commit(lead, &bars.o_full[i]);
          }
        }
        if (ok) {
          commit(lead, &bars.v_empty[s]);
          if (j + 1 < n) commit(lead, &bars.k_empty[s1]);
        }
      }
      failed = !ok;
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    const int i = warp >> 2;  // tile
    if (i < tiles) {
      const int row = threadIdx.x & 127;
      f = t.f0 + 128 * i + row;
      const int tok = fast_div(f, p.group_div), h = kvh * p.group + f - tok * p.group, pos = t.past + tok;
      const float slope = a.slopes && f < last ? a.slopes[h] * kLog2e : 0.f;
      const uint32_t lanes = uint32_t(32 * (warp & 3)) << 16;
      const uint32_t ts = tmem + lanes + s_col + 128 * i, to = tmem + lanes + o_col + D * i;
      float m = -INFINITY;  // reference maximum of the row, log2
      for (int j = 0; j < n; ++j) {
        if (!warp_wait(&bars.s_full[i], j & 1)) { failed = true; break; }
        fence_after();
        float x[PT_N];
#pragma unroll
        for (int c = 0; c < PT_N / 32; ++c) ld32(ts + 32 * c, reinterpret_cast<uint32_t*>(x) + 32 * c);
        ld_wait();
        const int base = blocks.base(j, PT_N);
        if constexpr (MOD) {
          if (p.a.softcap > 0.f) {
#pragma unroll
            for (int c = 0; c < PT_N; ++c) x[c] = score_log2<true>(x[c], p);
          } else {
#pragma unroll
            for (int c = 0; c < PT_N; ++c) x[c] *= p.scale_log2;
          }
          if (a.slopes) {
#pragma unroll
            for (int c = 0; c < PT_N; ++c) x[c] -= slope * fabsf(float(pos - base - c));
          }
        }
        if (!seen_by_all(base)) {
#pragma unroll
          for (int c = 0; c < PT_N; ++c) {
            const int jj = base + c;
            if (!(jj < t.len && row_sees(p, t, pos, jj))) x[c] = -INFINITY;
          }
        }
        float mxs[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
        for (int c = 4; c < PT_N - 4; c += 8)
#pragma unroll
          for (int e = 0; e < 4; ++e) mxs[e] = max3(mxs[e], x[c + e], x[c + 4 + e]);
#pragma unroll
        for (int e = 0; e < 4; ++e) mxs[e] = fmaxf(mxs[e], x[PT_N - 4 + e]);
        float mx = fmaxf(max3(mxs[0], mxs[1], mxs[2]), mxs[3]);
        if constexpr (!MOD) mx *= p.scale_log2;  // positive: rounding keeps the order
        float factor = 1.f;
        if (mx > m + PT_LAG || (j == 0 && mx > m)) {
          factor = m == -INFINITY ? 0.f : ex2(m - mx);
          m = mx;
        }
        if (__any_sync(~0u, factor != 1.f)) {
          l *= factor;
          if (j > 0) {
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
              uint32_t o[32];
              ld32(to + 32 * c, o);
              ld_wait();
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * factor);
              st32(to + 32 * c, o);
            }
          }
        }
        const float z = m == -INFINITY ? 0.f : -m;
        uint32_t w[PT_N / 2];
        uint64_t part[2] = {pair(l, 0.f), pair(0.f, 0.f)};
        const uint64_t z2 = pair(z, z), scale2 = pair(p.scale_log2, p.scale_log2);
#pragma unroll
        for (int c = 0; c < PT_N; c += 2) {
          float2 y;
          if constexpr (MOD) y = split(add2(pair(x[c], x[c + 1]), z2));
          else y = split(fma2(pair(x[c], x[c + 1]), scale2, z2));
          y.x = ex2(y.x);
          y.y = ex2(y.y);
          part[(c >> 1) & 1] = add2(part[(c >> 1) & 1], pair(y.x, y.y));
          w[c / 2] = pack2<DT>(y.x, y.y);
        }
        const float2 sum = split(add2(part[0], part[1]));
        l = sum.x + sum.y;
        st32(ts, w);
        st32(ts + 32, w + 32);
        st_wait();
        fence_before();
        mbar_arrive(&bars.p_ready[i]);
      }
      if (n > 0 && !failed && !warp_wait(&bars.o_full[i], 0)) failed = true;
      fence_after();
      const float inv = l == 0.f ? 0.f : 1.0f / l;
      T* out = static_cast<T*>(a.out) + int64_t(t.first + tok) * a.o_stride_t + h * a.o_stride_h;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32], w[16];
        if (n > 0) {
          ld32(to + 32 * c, o);
          ld_wait();
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0u;
        }
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          const float u = __uint_as_float(o[e]) * inv, v = __uint_as_float(o[e + 1]) * inv;
          odd += (u + v) * 0.f;
          w[e / 2] = pack2<DT>(u, v);
        }
        if (f < last && !failed) {
#pragma unroll
          for (int e = 0; e < 4; ++e) reinterpret_cast<uint4*>(out + 32 * c)[e] = make_uint4(w[4 * e], w[4 * e + 1], w[4 * e + 2], w[4 * e + 3]);
        }
      }
      if (a.lse && f < last) a.lse[int64_t(t.first + tok) * a.n_q_heads + h] = (m + log2f(l)) * kLn2;
    }
  }
  if (failed) atomicOr(&g_prefill_fault, 1u);
  fence_before();
  __syncthreads();
  if (warp == PT_MMA_WARP) {
    fence_after();
    dealloc(bars.tmem, PT_COLS);
  }
  if (warp < PT_LOAD_WARP && bars.special && (warp >> 2) < tiles) {
    uint32_t redo = __ballot_sync(~0u, odd != 0.f && l == l && f < last);
    for (; redo; redo &= redo - 1) exact_row(p, t, kvh, __shfl_sync(~0u, f, __ffs(redo) - 1));
  }
}

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &ptr, 12000, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
  });
  return fn;
}

// A cache as [pages][slots][heads][channels] for boxes of 64 channels by one head by `box` slots of a page.
bool encode(CUtensorMap* map, const smaq_paged_args& a, const void* cache, int box) {
  auto fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[4] = {cuuint64_t(a.head_dim), cuuint64_t(a.n_kv_heads), cuuint64_t(a.page_size), cuuint64_t(a.n_pages)};
  auto bytes = [](int64_t stride, int64_t n) { return cuuint64_t(n > 1 ? stride * 2 : 16); };  // of one element: not used
  const cuuint64_t strides[3] = {bytes(a.c_stride_h, a.n_kv_heads), bytes(a.c_stride_slot, a.page_size), bytes(a.c_stride_page, a.n_pages)};
  for (const cuuint64_t s : strides)
    if (s == 0 || s >= (cuuint64_t(1) << 40)) return false;
  const cuuint32_t shape[4] = {64u, 1u, cuuint32_t(box), 1u}, step[4] = {1u, 1u, 1u, 1u};
  return fn(map, a.dtype == SMAQ_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(cache), dims,
            strides, shape, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <class DT, int D>
int launch(const PagedParams& p, cudaStream_t st) {
  PtParams pt;
  pt.p = p;
  const smaq_paged_args& a = p.a;
  // boxes tile a block of 128 tokens when a page is 8 to 128 slots and divides it, or is a multiple of it
  pt.box = a.page_size < PT_N ? a.page_size : PT_N;
  pt.tma = a.page_size >= 8 && (a.page_size < PT_N ? PT_N % a.page_size : a.page_size % PT_N) == 0 && a.n_pages > 0 && a.n_pages < (int64_t(1) << 31) &&
           encode(&pt.k, a, a.k_cache, pt.box) && encode(&pt.v, a, a.v_cache, pt.box);
  const bool mod = p.a.softcap > 0.f || p.a.slopes || !(p.a.scale > 0.f);
  auto kern = mod ? prefill_tc_kernel<DT, D, true> : prefill_tc_kernel<DT, D, false>;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, PtCfg<D>::SMEM);
  if (e != cudaSuccess) return cuda_status(e, "paged_prefill attr");
  const int64_t tiles = (p.a.n_rows * p.group + PT_ROWS - 1) / PT_ROWS + p.a.batch;
  if (tiles * a.n_kv_heads >= (int64_t(1) << 31)) return fail(SMAQ_ERR_UNSUPPORTED, "paged_prefill: too many rows");
  kern<<<unsigned(tiles * a.n_kv_heads), PT_THREADS, PtCfg<D>::SMEM, st>>>(pt);
  return cuda_status(cudaGetLastError(), "paged_prefill");
}

}  // namespace

bool prefill_tc_eligible(const smaq_paged_args& a) {
  return a.dtype != SMAQ_F32 && (a.head_dim == 64 || a.head_dim == 128) && paged_aligned(a);
}

int launch_prefill_tc(const PagedParams& p, cudaStream_t st) {
  if (p.a.dtype == SMAQ_BF16) return p.a.head_dim == 64 ? launch<BF16, 64>(p, st) : launch<BF16, 128>(p, st);
  return p.a.head_dim == 64 ? launch<F16, 64>(p, st) : launch<F16, 128>(p, st);
}

}  // namespace smaq

extern "C" int smaq_prefill_status(void* stream) {
  cudaError_t e = cudaStreamSynchronize(static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return smaq::cuda_status(e, "prefill status: stream");
  unsigned int word = 0, zero = 0;
  e = cudaMemcpyFromSymbol(&word, smaq::g_prefill_fault, sizeof(word));
  if (e == cudaSuccess && word) e = cudaMemcpyToSymbol(smaq::g_prefill_fault, &zero, sizeof(zero));
  if (e != cudaSuccess) return smaq::cuda_status(e, "prefill status: read");
  if (word) return smaq::fail(SMAQ_ERR_DEVICE, "prefill: a bounded device wait of the tensor-core kernel ran out");
  return SMAQ_OK;
}
