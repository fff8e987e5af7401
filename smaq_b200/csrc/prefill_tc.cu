// Prefill attention on the 5th-generation tensor cores (bf16 / fp16, head_dim 64, 128 and 256).
//
// A CTA holds 256 rows (tokens times grouped heads, paged_prefill.cuh) as two tiles of 128 and walks blocks of 128
// tokens.  For each tile and block S = Q K^T goes to tensor memory, a warpgroup turns it into weights P there, and
// O += P V reads P from tensor memory.  The two tiles take turns: while one is in its softmax the tensor cores work for
// the other.
//   warps 0-7, 8-15  softmax of tile 0, 1: a thread has one half of a row's scores and goes over them twice, 32 columns at a time
//                    (maximum, weights); the halves' maxima meet in shared memory.  (One thread a row with its 128 scores in
//                    registers has half the warps to hide latencies with: measured together, 541 us against 539 at 8192
//                    tokens, 728 against 712 capped.)
//   warps 16-18      copies of keys and values, by TMA in boxes of a page (where a block has tokens that no row sees, the values'
//                    rows are cleared), or by cp.async of 16 bytes for page sizes that do not tile a block (such tokens are
//                    written as zeros), both in the 128-byte swizzled operand layout; the softmax threads load the queries;
//   warp 19          issues all products.
// Tensor memory: S0 S1 (128 columns each), O0 O1 (head_dim each); P overwrites its S.  The product for the next S of a tile is
// issued right behind the product that reads its P, and its completion also says that O is at rest: a softmax warp may
// then rescale O, which it does only when a row's maximum grew by more than 2^8, in fp16 2^3 (the reference of a row lags by
// at most that, so weights stay below 2^8 in bf16 and 2^15 in fp16).
// At head_dim 256 there is room for one tile (128 rows, half the softmax warps): S0 and S1 are then blocks of even and odd
// number, the next block's scores are computed during this block's softmax, and O is waited for by itself.
// Weights are rounded once, to the cache's type, as the operand of the second product; the sums are of the unrounded ones.
// Two parts a weight, as in decode, would double that product and leave no tensor memory for a second tile.  Against 64 bits
// an answer is off by 0.0018 to 0.0020 of its size in bf16 and 0.0003 in fp16, of which the output's own rounding is 0.0016
// and 0.0002.
// Few rows with long walks: several CTAs share a tile's walk and prefill_join_kernel adds their parts in order.
// Products and exponentials take 2048 cycles a block each, side by side, of about 3300 in all; the rest is the way from a
// block's scores to its weights, which two tiles do not hide.  8192 tokens at 32/8 heads of 128: 522 to 527 us on the device
// in short runs (1050 TFLOP/s, 63% of what a library product reaches there), 586 to 605 a call in long ones (915 to 938),
// under the power cap.
// Every wait is bounded; one that runs out sets g_prefill_fault, and its rows come out as NaN.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <atomic>

#include "paged_prefill.cuh"
#include "prefill_tc.cuh"
#include "tcgen05.cuh"

namespace smaq {

namespace {

using namespace tc5;

__device__ unsigned int g_prefill_fault;

constexpr int PT_SPLIT = 2;               // softmax threads a row
constexpr int PT_TW = 4 * PT_SPLIT;       // softmax warps a tile
constexpr int PT_N = 128;                 // tokens a block
constexpr int PT_LOADERS = 96;            // three warps of copies
constexpr int PJ_ROWS = 32;               // rows a CTA of the join
// Tiles a CTA: tensor memory has room for the scores and accumulators of two at head_dim 128, of one at 256.
__host__ __device__ constexpr int pt_tiles(int D) { return D == 256 ? 1 : 2; }
__host__ __device__ constexpr int pt_rows(int D) { return 128 * pt_tiles(D); }
__host__ __device__ constexpr int pt_threads(int D) { return 32 * (PT_TW * pt_tiles(D) + 4); }
constexpr uint32_t PT_COLS = 512;
// log2: how far a row's maximum may grow above its reference before O is rescaled.  In fp16 the weights have room for 2^15
// (paged.cuh): the reference lies 2^12 below the maximum it was taken from, which leaves 2^3.
template <class DT>
constexpr float PT_LAG = DT::code == SMAQ_F16 ? 3.0f : 8.0f;
template <class DT>
constexpr float PT_UP = kUp<DT> > 0.f ? kUp<DT> - PT_LAG<DT> : 0.0f;

template <int D>
struct PtCfg {
  static constexpr int TILES = pt_tiles(D);
  static constexpr int TILE = 128 * D * 2;              // bytes: 128 rows of queries, keys or values
  static constexpr int STAGES = D == 256 ? 1 : 2;
  static constexpr int SMEM = TILES * TILE + 2 * STAGES * TILE + 1024;
};

struct PtParams {
  PagedParams p;
  int tma;         // keys and values come through the tensor maps where a block's pages allow it
  int box;         // slots a box: page_size, at most PT_N
  int splits;      // CTAs that share a tile's walk, at most
  uint32_t spin;   // polls before a wait gives up
  float* parts;    // [tile][KV head][split]: accumulators [rows][D], maxima, sums, whether a special value was met
  CUtensorMap k, v;
};
__host__ __device__ constexpr int64_t part_floats(int D) { return int64_t(pt_rows(D)) * (D + 2) + 4; }
// Splits of a walk of n blocks: two blocks each at least.
__device__ __forceinline__ int splits_of(int n, int most) { return max(1, min(most, n / 2)); }

struct PtBars {
  uint64_t q_full, v_part, k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_ready[2], o_step, o_full[2], drained;
  uint32_t tmem;
  int special;
  // the tile and its walk: read from here where needed, the softmax has no registers for them
  PrefillTile t;
  PrefillBlocks blocks;
  int least, most;          // first and last row's position
  float row[2][2][2][128];  // [turn][tile][half]: row maxima, at the end row sums
  int fail[2][2][4];        // [turn][tile][rows]: a wait of one of the two warps that share rows ran out: both stop at that turn's meeting
};

__device__ __forceinline__ void named_bar(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }

enum { PT_PLAIN = 0, PT_CAP = 1, PT_ANY = 2 };  // scores: scaled by a positive factor; capped; everything else
// PT_CAP's tanh is that of caps up to kCapNear; the series beside it would be half of its softmax again.
// Of every PT_OF pairs of exponentials so many come from the polynomial, the others from the special-function unit,
// which alone would need as long as the products.  At 8192 tokens and 32/8 heads 0, 1, 2, 3 of 8 took 515, 514, 533,
// 548 us; a capped score takes two exponentials and a reciprocal: (4, 2), (5, 2), (5, 3), (4, 1), (6, 3) of 8 for (tanh,
// weight) took 673, 666, 676, 684, 689 us on chunks of 64/8 heads behind 8K tokens.
constexpr int PT_POLY = 1, PT_POLY_CAP = 5, PT_POLY_EXP = 2;
constexpr int PT_OF = 8;

// 2^x of PT_OF pairs, POLY of them by the polynomial.
template <int DEG, int POLY>
__device__ __forceinline__ void exp2_group(uint64_t (&x)[PT_OF]) {
  if constexpr (POLY > 0) {
    uint64_t y[POLY];
#pragma unroll
    for (int i = 0; i < POLY; ++i) y[i] = x[i];
    exp2_poly<DEG>(y);
#pragma unroll
    for (int i = 0; i < POLY; ++i) x[i] = y[i];
  }
#pragma unroll
  for (int i = POLY; i < PT_OF; ++i) {
    const float2 v = split(x[i]);
    x[i] = pair(ex2(v.x), ex2(v.y));
  }
}

template <class DT, int D, int MODE>
__global__ void __launch_bounds__(pt_threads(D), 1) prefill_tc_kernel(const __grid_constant__ PtParams pt) {
  using T = typename DT::T;
  const PagedParams& p = pt.p;
  constexpr int TILES = PtCfg<D>::TILES, ROWS = pt_rows(D), LOAD_WARP = PT_TW * TILES, MMA_WARP = LOAD_WARP + 3;
  constexpr int TILE = PtCfg<D>::TILE, STAGES = PtCfg<D>::STAGES, CH = D / 8, GROUP = 8 * D * 2;  // GROUP: 8 rows, 64-channel atoms side by side
  constexpr uint32_t ID_S = idesc(DT::code == SMAQ_BF16, PT_N, false), ID_O = idesc(DT::code == SMAQ_BF16, D, true);
  extern __shared__ uint8_t smem_raw[];
  __shared__ PtBars bars;
  __shared__ int sums[pt_threads(D) / 32];
  const smaq_paged_args& a = p.a;
  const uint32_t base_raw = smem_u32(smem_raw), pad = (1024u - (base_raw & 1023u)) & 1023u;
  uint8_t* smem = smem_raw + pad;
  const uint32_t qs = base_raw + pad, ks = qs + TILES * TILE, vs = ks + STAGES * TILE;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, share = int(blockIdx.x % unsigned(pt.splits));
  const int kvh = int(blockIdx.x / unsigned(pt.splits) % unsigned(a.n_kv_heads)), tile = int(blockIdx.x / unsigned(pt.splits * a.n_kv_heads));
  pdl_launch_dependents();

  int n, first_block, tiles, last;  // blocks of this CTA's share, the first of them
  bool alone;                      // the share is the whole walk
  {
    const PrefillTile t = find_tile<pt_threads(D)>(p, tile, ROWS, true, sums, &bars.t);
    const PrefillBlocks blocks(t, PT_N);
    const int shares = t.rows ? splits_of(blocks.count, pt.splits) : 0;
    if (share >= shares) {  // also where the number of tiles that the host allows for exceeds theirs
      if (share == 0) write_padding(p, kvh, tile, int(gridDim.x / unsigned(pt.splits * a.n_kv_heads)));
      return;
    }
    first_block = int(int64_t(blocks.count) * share / shares);
    n = int(int64_t(blocks.count) * (share + 1) / shares) - first_block;
    alone = shares == 1;
    tiles = t.rows > 128 ? 2 : 1;
    last = t.f0 + t.rows;
    if (threadIdx.x == 0) {
      bars.blocks = blocks;
      bars.least = t.past + fast_div(t.f0, p.group_div);
      bars.most = t.past + fast_div(last - 1, p.group_div);
    }
  }
  const PrefillTile& t = bars.t;
  const PrefillBlocks& blocks = bars.blocks;

  if (threadIdx.x == 0) {
    mbar_init(&bars.q_full, TILES * PT_TW);
    mbar_init(&bars.o_step, 1);
    mbar_init(&bars.drained, 1);
    mbar_init(&bars.v_part, PT_LOADERS / 32);  // one arrival a copying warp: a phase ends only when all have passed the last
    for (int s = 0; s < 2; ++s) {
      mbar_init(&bars.k_full[s], PT_LOADERS);
      mbar_init(&bars.v_full[s], PT_LOADERS);
      mbar_init(&bars.k_empty[s], 1);
      mbar_init(&bars.v_empty[s], 1);
      mbar_init(&bars.s_full[s], 1);
      mbar_init(&bars.p_ready[s], PT_TW);
      mbar_init(&bars.o_full[s], 1);
    }
    bars.special = 0;
    for (int i = 0; i < 16; ++i) bars.fail[i >> 3][i >> 2 & 1][i & 3] = 0;
    fence_mbar_init();
  }
  if (warp == MMA_WARP) alloc(&bars.tmem, PT_COLS);
  fence_before();
  __syncthreads();
  fence_after();
  constexpr uint32_t tmem = 0;  // all 512 columns are this CTA's: the allocation starts at 0
  constexpr uint32_t s_col = 0, o_col = 256;  // S of tile i (one tile: of blocks of parity i) at s_col + 128 i, O at o_col + D i
  bool failed = false;
  // The whole warp waits, and gives up together.
  auto warp_wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(~0u, mbar_wait(bar, parity, pt.spin)); };

  // a row's chunk of eight channels in an operand
  auto at = [](int r, int ch) { return uint32_t((r >> 3) * GROUP + (ch >> 3) * 1024 + (r & 7) * 128 + (((ch & 7) ^ (r & 7)) << 4)); };
  auto base_of = [&](int j) { return blocks.base(first_block + j, PT_N); };
  auto seen_by_all = [&](int base) {
    return base + PT_N <= t.prefix || (base + PT_N <= bars.least + 1 && (a.window == 0 || base > bars.most - a.window));
  };
  float odd = 0.f, l = 0.f;  // softmax threads: NaN where an output is not finite; sum of weights
  int f = 0;

  if (warp >= LOAD_WARP) {
    if constexpr (TILES == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");  // 128 x 64 + 512 x 104 = 640 x 96, the launch's
    if (warp < MMA_WARP) {
      // ---- copies
      const int w = warp - LOAD_WARP, tid = threadIdx.x - LOAD_WARP * 32;
      const uint32_t lead = elect_one();
      const int32_t* table = a.block_table + t.b * a.table_stride;
      // By TMA a block comes in boxes of one page (or 128 slots of it), the warps in turn; a box without a token that some
      // row sees is left out.  (Issued by the lanes of one warp side by side, boxes cost about 150 cycles each.)
      const int per = PT_N / pt.box;
      auto needed = [&](int k) {  // this lane's box of block k
        const int b = base_of(k) + lane * pt.box;
        return pt.tma && k < n && lane < per && (b < t.prefix || (b + pt.box > t.lo && b < t.hi));
      };
      auto page_of = [&](int k) {
        if (!needed(k)) return 0;
        const int64_t blk = fast_div(base_of(k) + lane * pt.box, p.page_div);
        return int(min(max(int64_t(__ldg(table + blk)), int64_t(0)), a.n_pages - 1));
      };
      int partial = 0;  // blocks whose values came through v_part
      // Blocks that come by cp.async: warp w brings rows r0 .. r0 + rows of every operand.
      const int r0 = w * 43, rows = min(43, PT_N - r0);
      // values of a block that some rows see in part: look for infinities and NaN in this warp's rows
      auto look_for_special = [&](int s) {
        bool odd_value = false;
        const uint8_t* stage = smem + (vs - qs) + s * TILE;
#pragma unroll 8
        for (int i = lane; i < rows * CH; i += 32) odd_value |= any_special<DT>(*reinterpret_cast<const uint4*>(stage + at(r0 + i / CH, i % CH)));
        if (odd_value) bars.special = 1;
      };
      auto fetch = [&](int j, int s, bool values, int page) {
        uint64_t* bar = values ? &bars.v_full[s] : &bars.k_full[s];
        const uint32_t dst = (values ? vs : ks) + s * TILE;
        const bool part = values && !seen_by_all(base_of(j));
        if (pt.tma) {
          // The scores of tokens that a row does not see are replaced whatever their keys are, but their values are multiplied
          // by zero.  A block that is not seen by all rows therefore has its values arrive at v_part: rows that nobody sees are
          // cleared and the others looked through before the products may have them, since from then on another warp may
          // fill the stage again.
          const uint32_t boxes = __ballot_sync(~0u, needed(j));
          uint64_t* here = part ? &bars.v_part : bar;
          if (tid == 0) mbar_arrive_expect_tx(here, __popc(boxes) * pt.box * D * 2);
          const int first = base_of(j), slot = per > 1 ? 0 : first - fast_div(first, p.page_div) * a.page_size;
          for (int b = w; b < per; b += MMA_WARP - LOAD_WARP) {
            const int pg = __shfl_sync(~0u, page, b);
            if (boxes >> b & 1) tma_5d(lead, dst + b * pt.box * (D * 2), values ? &pt.v : &pt.k, kvh * int(a.c_stride_h), 0, 0, slot >> 3, pg, here);
          }
          if (part) {
            if (w > 0 && lane == 0) mbar_arrive(here);
            if (!warp_wait(here, partial++ & 1)) failed = true;
            const int pre = t.prefix - first, lo = t.lo - first, hi = t.hi - first;
            if (pre < PT_N && (lo > 0 || hi < PT_N)) {
#pragma unroll 4
              for (int i = lane; i < rows * CH; i += 32)
                if (const int r = r0 + i / CH; r >= pre && (r < lo || r >= hi)) *reinterpret_cast<uint4*>(smem + (dst - qs) + at(r0 + i / CH, i % CH)) = make_uint4(0, 0, 0, 0);
              __syncwarp();
            }
            look_for_special(s);
            fence_proxy_async_smem();
            mbar_arrive(bar);
          } else if (tid != 0) {
            mbar_arrive(bar);
          }
          return;
        }
        const T* cache = static_cast<const T*>(values ? a.v_cache : a.k_cache);
        auto offset = [&](int r) {
          const int tok = base_of(j) + r0 + r;
          return r < rows && tile_sees(t, tok) ? token_offset(p, table, tok) + kvh * a.c_stride_h : int64_t(-1);
        };
        const int64_t off0 = offset(lane), off1 = offset(lane + 32);
#pragma unroll 4
        for (int i0 = 0; i0 < 44 * CH; i0 += 32) {
          const int r = (i0 + lane) / CH, ch = (i0 + lane) % CH;
          const int64_t lo = __shfl_sync(~0u, off0, r & 31), hi = __shfl_sync(~0u, off1, r & 31);
          const int64_t off = r < 32 ? lo : hi;
          if (r < rows) cp_async16(dst + at(r0 + r, ch), cache + (off < 0 ? 0 : off) + ch * 8, off < 0 ? 0u : 16u);
        }
        cp_async_commit();
        cp_async_wait<0>();
        if (part) {
          __syncwarp();  // the other lanes' copies too
          look_for_special(s);
        }
        fence_proxy_async_smem();
        mbar_arrive(bar);
      };
      int page = page_of(0), k_sent = 0, v_sent = 0;
      for (int j = 0; j < n; ++j) {
        const int s = j % STAGES;
        const uint32_t ph = uint32_t((j / STAGES) & 1) ^ 1u;
        const int next = page_of(j + 1);
        if (!warp_wait(&bars.k_empty[s], ph)) { failed = true; break; }
        fetch(j, s, false, page);
        ++k_sent;
        if (!warp_wait(&bars.v_empty[s], ph)) { failed = true; break; }
        fetch(j, s, true, page);
        ++v_sent;
        if (failed) break;
        page = next;
      }
      if (failed) {  // copies in flight land before the block leaves
        for (int j = max(k_sent - STAGES, 0); j < k_sent; ++j) mbar_drain(&bars.k_full[j % STAGES], (j / STAGES) & 1);
        for (int j = max(v_sent - STAGES, 0); j < v_sent; ++j) mbar_drain(&bars.v_full[j % STAGES], (j / STAGES) & 1);
        if (partial > 0) mbar_drain(&bars.v_part, (partial - 1) & 1);
      }
    } else if (warp == MMA_WARP && n > 0) {
      // ---- products
      const uint32_t lead = elect_one();
      auto scores = [&](int i, int j) {
        const uint32_t q = qs + (TILES == 2 ? i * TILE : 0), k = ks + (j % STAGES) * TILE;
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
          const uint32_t at = uint32_t((c >> 2) * 1024 + (c & 3) * 32);
          mma_ss(lead, tmem + s_col + 128 * i, desc(q + at, GROUP, 16), desc(k + at, GROUP, 16), ID_S, c > 0);
        }
        commit(lead, &bars.s_full[i]);
      };
      auto values = [&](int i, int j) {
        const uint32_t v = vs + (j % STAGES) * TILE;
#pragma unroll
        for (int c = 0; c < PT_N / 16; ++c)
          mma_ts(lead, tmem + o_col + (TILES == 2 ? D * i : 0), tmem + s_col + 128 * i + 64 * (c >> 2) + 8 * (c & 3), desc(v + c * 2 * GROUP, GROUP, 1024),
                 ID_O, (j > 0) | (c > 0));
      };
      bool ok = warp_wait(&bars.q_full, 0) && warp_wait(&bars.k_full[0], 0);
      if (ok) {
        fence_after();
        for (int i = 0; i < tiles; ++i) scores(i, 0);
        commit(lead, &bars.k_empty[0]);
      }
      for (int j = 0; ok && j < n; ++j) {
        const int s = j % STAGES, s1 = (j + 1) % STAGES;
        if constexpr (TILES == 1) {
          // the next block's scores, in the other buffer, keep the tensor cores busy during this block's softmax
          if (j + 1 < n) {
            ok = warp_wait(&bars.k_full[s1], ((j + 1) / STAGES) & 1);
            if (!ok) break;
            fence_after();
            scores((j + 1) & 1, j + 1);
            commit(lead, &bars.k_empty[s1]);
          }
          ok = warp_wait(&bars.v_full[s], (j / STAGES) & 1) && warp_wait(&bars.p_ready[j & 1], (j >> 1) & 1);
          if (!ok) break;
          fence_after();
          values(j & 1, j);
          commit(lead, &bars.o_step);
          commit(lead, &bars.v_empty[s]);
          if (j + 1 == n) commit(lead, &bars.o_full[0]);
          continue;
        }
        ok = warp_wait(&bars.v_full[s], (j / STAGES) & 1);
        for (int i = 0; ok && i < tiles; ++i) {
          ok = warp_wait(&bars.p_ready[i], j & 1);
          if (!ok) break;
          fence_after();
          values(i, j);
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
      if (failed) {  // products in flight end before their tensor memory is given back
        commit(lead, &bars.drained);
        mbar_drain(&bars.drained, 0);
      }
    }
  } else {
    if constexpr (TILES == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");  // one tile: 384 threads have 168 anyway
    // ---- queries
    for (int i = threadIdx.x; i < tiles * 128 * CH; i += LOAD_WARP * 32) {
      const int r = i / CH, ch = i % CH, fr = t.f0 + r, tok = fast_div(fr, p.group_div);
      const bool live = r < t.rows;
      const T* src = static_cast<const T*>(a.q) + (live ? (t.first + tok) * a.q_stride_t + (kvh * p.group + fr - tok * p.group) * a.q_stride_h + ch * 8 : 0);
      cp_async16(qs + at(r, ch), src, live ? 16u : 0u);
    }
    cp_async_commit();
    cp_async_wait<0>();
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(&bars.q_full);
    constexpr int C = PT_N / PT_SPLIT;                  // columns a thread
    const int i = warp / PT_TW, half = (warp >> 2) & 1;  // tile, half of the columns
    if (i < tiles) {
      const int row = 32 * (warp & 3) + lane, meet = 2 + i * 4 + (warp & 3);  // barrier of the two warps that share these rows
      f = t.f0 + 128 * i + row;
      const int tok = fast_div(f, p.group_div), h = kvh * p.group + f - tok * p.group, pos = t.past + tok;
      const float slope = a.slopes && f < last ? a.slopes[h] * kLog2e : 0.f;
      const uint32_t lanes = uint32_t(32 * (warp & 3)) << 16;
      const uint32_t to = tmem + lanes + o_col + D * i + half * (D / PT_SPLIT);
      float m = -INFINITY;  // reference of the row, log2
      for (int j = 0; j < n; ++j) {
        const int base = base_of(j) + half * C;
        const bool part = !seen_by_all(base - half * C);
        const int buf = TILES == 2 ? i : j & 1;  // of the scores
        const uint32_t ts = tmem + lanes + s_col + 128 * buf;
        if (!warp_wait(&bars.s_full[buf], (TILES == 2 ? j : j >> 1) & 1)) bars.fail[j & 1][i][warp & 3] = 1;
        fence_after();
        // Two passes over the scores, 32 columns at a time, so that they need not stay in registers: the first
        // finds the maximum and puts capped, biased or masked scores back, the second makes the weights.
        float mx = -INFINITY;
        float x[32];
#pragma unroll
        for (int q = 0; q < C / 32; ++q) {
          ld32(ts + half * C + 32 * q, reinterpret_cast<uint32_t*>(x));
          ld_wait();
          const int b = base + 32 * q;
          if constexpr (MODE == PT_CAP) {
            const uint64_t in2 = pair(p.cap_in, p.cap_in), out2 = pair(-2.0f * p.cap_log2, -2.0f * p.cap_log2), cap2 = pair(p.cap_log2, p.cap_log2);
#pragma unroll
            for (int c = 0; c < 32; c += 2 * PT_OF) {  // cap tanh, as score_log2 far from zero
              uint64_t y[PT_OF];
#pragma unroll
              for (int e = 0; e < PT_OF; ++e) {
                y[e] = mul2(pair(x[c + 2 * e], x[c + 2 * e + 1]), in2);
                if (e < PT_POLY_CAP) {  // the polynomial's range: tanh is 1 long before
                  float2 v = split(y[e]);
                  asm("min.NaN.f32 %0, %0, %1;" : "+f"(v.x) : "f"(126.0f));
                  asm("min.NaN.f32 %0, %0, %1;" : "+f"(v.y) : "f"(126.0f));
                  y[e] = pair(v.x, v.y);
                }
              }
              exp2_group<5, PT_POLY_CAP>(y);
#pragma unroll
              for (int e = 0; e < PT_OF; ++e) {
                const float2 v = split(add2(y[e], pair(1.0f, 1.0f)));
                const float2 u = split(fma2(pair(rcp_approx(v.x), rcp_approx(v.y)), out2, cap2));
                x[c + 2 * e] = u.x;
                x[c + 2 * e + 1] = u.y;
              }
            }
          } else if constexpr (MODE == PT_ANY) {
            if (p.a.softcap > 0.f) {
#pragma unroll
              for (int c = 0; c < 32; ++c) x[c] = score_log2<CAP_ANY>(x[c], p);
            } else {
#pragma unroll
              for (int c = 0; c < 32; ++c) x[c] *= p.scale_log2;
            }
            if (a.slopes) {
#pragma unroll
              for (int c = 0; c < 32; ++c) x[c] -= slope * fabsf(float(pos - b - c));
            }
          }
          if (part) {
            const int upper = min(pos + 1, t.len) - b;
            if (t.prefix <= base && (a.window == 0 || base - half * C > bars.most - a.window)) {  // cut by the row's own position alone
#pragma unroll
              for (int c = 0; c < 32; ++c) x[c] = c < upper ? x[c] : -INFINITY;
            } else {
              const int lower = a.window ? pos - a.window + 1 - b : 0, pre = t.prefix - b;
#pragma unroll
              for (int c = 0; c < 32; ++c) x[c] = c < pre || (c >= lower && c < upper) ? x[c] : -INFINITY;
            }
          }
          if (MODE != PT_PLAIN || part) st32(ts + half * C + 32 * q, reinterpret_cast<const uint32_t*>(x));
          float mxs[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
          for (int c = 4; c < 28; c += 8)
#pragma unroll
            for (int e = 0; e < 4; ++e) mxs[e] = max3(mxs[e], x[c + e], x[c + 4 + e]);
          mx = max3(mx, max3(mxs[0], mxs[1], mxs[2]), max3(mxs[3], x[28], x[29]));
          mx = max3(mx, x[30], x[31]);
        }
        if constexpr (MODE == PT_PLAIN) mx *= p.scale_log2;  // positive: rounding keeps the order
        if (MODE != PT_PLAIN || part) st_wait();
        bars.row[j & 1][i][half][row] = mx;
        named_bar(meet, 64);
        mx = fmaxf(mx, bars.row[j & 1][i][half ^ 1][row]);
        if (*reinterpret_cast<volatile int*>(&bars.fail[j & 1][i][warp & 3])) { failed = true; break; }
        mx -= PT_UP<DT>;
        float factor = 1.f;
        if (mx > m + PT_LAG<DT> || (j == 0 && mx > m)) {
          factor = m == -INFINITY ? 0.f : ex2(m - mx);
          m = mx;
        }
        if (__any_sync(~0u, factor != 1.f)) {
          l *= factor;
          if (j > 0) {
            if constexpr (TILES == 1) {  // these scores were multiplied before the last block's values
              if (!warp_wait(&bars.o_step, (j - 1) & 1)) bars.fail[(j + 1) & 1][i][warp & 3] = 1;
              fence_after();
            }
#pragma unroll 1  // cold: unrolled, its code costs the first pass 10 us of 519
            for (int c = 0; c < D / PT_SPLIT / 32; ++c) {
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
        uint64_t part2[2] = {pair(l, 0.f), pair(0.f, 0.f)};
        const uint64_t z2 = pair(z, z), scale2 = pair(p.scale_log2, p.scale_log2);
#pragma unroll
        for (int q = 0; q < C / 32; ++q) {
          uint32_t w[16];
          ld32(ts + half * C + 32 * q, reinterpret_cast<uint32_t*>(x));
          ld_wait();
#pragma unroll
          for (int c = 0; c < 32; c += 2 * PT_OF) {
            uint64_t y[PT_OF];
#pragma unroll
            for (int e = 0; e < PT_OF; ++e) {
              const uint64_t v = pair(x[c + 2 * e], x[c + 2 * e + 1]);
              y[e] = MODE == PT_PLAIN ? fma2(v, scale2, z2) : add2(v, z2);
            }
            exp2_group<4, MODE == PT_CAP ? PT_POLY_EXP : PT_POLY>(y);
#pragma unroll
            for (int e = 0; e < PT_OF; ++e) {
              part2[e & 1] = add2(part2[e & 1], y[e]);
              const float2 v = split(y[e]);
              w[c / 2 + e] = pack2<DT>(v.x, v.y);
            }
          }
          st16(ts + half * C + 16 * q, w);  // over scores that this thread has read
        }
        const float2 sum = split(add2(part2[0], part2[1]));
        l = sum.x + sum.y;
        st_wait();
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.p_ready[buf]);
      }
      if (n > 0 && !failed && !warp_wait(&bars.o_full[i], 0)) failed = true;
      fence_after();
      bars.row[n & 1][i][half][row] = l;
      named_bar(meet, 64);
      l += bars.row[n & 1][i][half ^ 1][row];
      failed |= *reinterpret_cast<volatile int*>(&bars.fail[n & 1][i][warp & 3]) != 0;
      if (failed) l = __int_as_float(0x7FC00000);  // a row whose wait ran out is NaN, here or from the join
      if (alone) {
        const float inv = l == 0.f ? 0.f : 1.0f / l;
        T* out = static_cast<T*>(a.out) + int64_t(t.first + tok) * a.o_stride_t + h * a.o_stride_h + half * (D / PT_SPLIT);
#pragma unroll 1
        for (int c = 0; c < D / PT_SPLIT / 32; ++c) {
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
          if (f < last) {
#pragma unroll
            for (int e = 0; e < 4; ++e) reinterpret_cast<uint4*>(out + 32 * c)[e] = make_uint4(w[4 * e], w[4 * e + 1], w[4 * e + 2], w[4 * e + 3]);
          }
        }
        if (a.lse && half == 0 && f < last) a.lse[int64_t(t.first + tok) * a.n_q_heads + h] = (m + log2f(l)) * kLn2;
      } else {
        float* part = pt.parts + int64_t(blockIdx.x) * part_floats(D);
        const int r = 128 * i + row;
#pragma unroll 1
        for (int c = 0; c < D / PT_SPLIT / 32; ++c) {
          uint32_t o[32];
          ld32(to + 32 * c, o);
          ld_wait();
          if (f < last) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              reinterpret_cast<uint4*>(part + r * D + half * (D / PT_SPLIT) + 32 * c)[e] = make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
          }
        }
        if (half == 0 && f < last) {
          part[ROWS * D + r] = m;
          part[ROWS * (D + 1) + r] = l;
        }
      }
    }
  }
  if (failed) atomicOr(&g_prefill_fault, 1u);
  fence_before();
  __syncthreads();
  if (warp == MMA_WARP) {
    fence_after();
    dealloc(bars.tmem, PT_COLS);
  }
  if (share == 0) write_padding(p, kvh, tile, int(gridDim.x / unsigned(pt.splits * a.n_kv_heads)));
  if (!alone) {
    if (threadIdx.x == 0) pt.parts[(int64_t(blockIdx.x) + 1) * part_floats(D) - 4] = bars.special ? 1.f : 0.f;
    return;
  }
  if (warp < LOAD_WARP && bars.special && warp / PT_TW < tiles) {
    uint32_t redo = __ballot_sync(~0u, odd != 0.f && l == l && f < last);
    for (; redo; redo &= redo - 1) exact_row(p, t, kvh, __shfl_sync(~0u, f, __ffs(redo) - 1));
  }
}

// ---------------------------------------------------------------- join of split walks
constexpr int PJ_THREADS = 256;

// PJ_ROWS rows of one tile and KV head, a warp each in turn: the shares in order.
template <class DT, int D>
__global__ void __launch_bounds__(PJ_THREADS) prefill_join_kernel(const __grid_constant__ PtParams pt) {
  using T = typename DT::T;
  constexpr int E = D / 32, ROWS = pt_rows(D);
  const PagedParams& p = pt.p;
  const smaq_paged_args& a = p.a;
  __shared__ int sums[PJ_THREADS / 32];
  __shared__ PrefillTile found;
  const int chunk = int(blockIdx.x % (ROWS / PJ_ROWS)), unit = int(blockIdx.x / (ROWS / PJ_ROWS));
  const int kvh = unit % a.n_kv_heads, tile = unit / a.n_kv_heads, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const PrefillTile t = find_tile<PJ_THREADS>(p, tile, ROWS, true, sums, &found);
  pdl_wait();  // every CTA waits, so this grid ends after the other
  const int shares = t.rows ? splits_of(PrefillBlocks(t, PT_N).count, pt.splits) : 0;
  if (shares < 2) return;
  const float* parts = pt.parts + int64_t(unit) * pt.splits * part_floats(D);
  bool special = false;
  for (int z = 0; z < shares; ++z) special |= parts[(z + 1) * part_floats(D) - 4] != 0.f;
  for (int r = chunk * PJ_ROWS + warp; r < min((chunk + 1) * PJ_ROWS, t.rows); r += PJ_THREADS / 32) {
    float m = -INFINITY, l = 0.f, o[E] = {};
    for (int z = 0; z < shares; ++z) m = fmaxf(m, parts[z * part_floats(D) + ROWS * D + r]);
    const float base = m == -INFINITY ? 0.f : m;
#pragma unroll 4
    for (int z = 0; z < shares; ++z) {
      const float* part = parts + z * part_floats(D);
      const float f = ex2(part[ROWS * D + r] - base);
      l += f * part[ROWS * (D + 1) + r];
      float x[E];
#pragma unroll
      for (int e = 0; e < E; e += 2) *reinterpret_cast<float2*>(x + e) = *reinterpret_cast<const float2*>(part + r * D + E * lane + e);
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] += f * x[e];
    }
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    const int f = t.f0 + r, tok = fast_div(f, p.group_div), h = kvh * p.group + f - tok * p.group;
    T* out = static_cast<T*>(a.out) + int64_t(t.first + tok) * a.o_stride_t + h * a.o_stride_h + E * lane;
    float odd = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      o[e] *= inv;
      odd += o[e] * 0.f;
    }
#pragma unroll
    for (int e = 0; e < E; e += 2) *reinterpret_cast<uint32_t*>(out + e) = pack2<DT>(o[e], o[e + 1]);
    if (a.lse && lane == 0) a.lse[int64_t(t.first + tok) * a.n_q_heads + h] = (m + log2f(l)) * kLn2;
    if (special && __any_sync(~0u, odd != 0.f) && l == l) {
      __syncwarp();
      exact_row(p, t, kvh, f);
    }
  }
}

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static const PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    const bool ok = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &ptr, 12000, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ok ? ptr : nullptr);
  }();
  return fn;
}

// A cache for boxes of `box` slots of a page by one head: channels of all heads in a row (a head begins at kvh *
// stride), eight slots, the 64-channel parts of a head, groups of eight slots, pages.  A box lands as it is
// multiplied: 8-row atoms, the parts of a head side by side.
bool encode(CUtensorMap* map, const smaq_paged_args& a, const void* cache, int box) {
  auto fn = encode_fn();
  if (!fn) return false;
  const int64_t row = (a.n_kv_heads - 1) * a.c_stride_h + 64;
  if (row < 64 || row >= (int64_t(1) << 31) || a.c_stride_slot <= 0 || (a.n_pages > 1 && a.c_stride_page <= 0)) return false;
  const cuuint64_t dims[5] = {cuuint64_t(row), 8, cuuint64_t(a.head_dim / 64), cuuint64_t(a.page_size / 8), cuuint64_t(a.n_pages)};
  const cuuint64_t strides[4] = {cuuint64_t(a.c_stride_slot) * 2, 128, cuuint64_t(a.c_stride_slot) * 16, cuuint64_t(a.n_pages > 1 ? a.c_stride_page * 2 : 16)};
  for (const cuuint64_t s : strides)
    if (s >= (cuuint64_t(1) << 40)) return false;
  const cuuint32_t shape[5] = {64u, 8u, cuuint32_t(a.head_dim / 64), cuuint32_t(box / 8), 1u}, step[5] = {1u, 1u, 1u, 1u, 1u};
  return fn(map, a.dtype == SMAQ_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 5, const_cast<void*>(cache), dims,
            strides, shape, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int64_t grid_tiles(int64_t n_rows, int batch, int group, int D) { return std::max<int64_t>(1, most_tiles(n_rows, batch, group, pt_rows(D))); }
// CTAs a tile: walks are shared where the tiles alone leave half of the GPU idle.  (The host does not know how long
// the walks are: a CTA without a share ends at once.)  16 rows of 32/8 heads behind 16K tokens: 227 -> 46 us.
int splits_for(int64_t units, int64_t max_tokens) {
  const int64_t idle = num_sms() / std::max<int64_t>(units, 1), worth = max_tokens / (2 * PT_N);  // two blocks a share
  return int(std::max<int64_t>(1, std::min<int64_t>(32, std::min(idle, worth))));
}

template <class DT, int D>
int launch(const PagedParams& p, cudaStream_t st) {
  PtParams pt;
  pt.p = p;
  const smaq_paged_args& a = p.a;
  // boxes tile a block of 128 tokens when a page is 8 to 128 slots and divides it, or is a multiple of it
  pt.box = a.page_size < PT_N ? a.page_size : PT_N;
  pt.tma = a.page_size >= 8 && (a.page_size < PT_N ? PT_N % a.page_size : a.page_size % PT_N) == 0 && a.n_pages > 0 && a.n_pages < (int64_t(1) << 31) &&
           a.n_kv_heads * a.c_stride_h < (int64_t(1) << 31) && encode(&pt.k, a, a.k_cache, pt.box) && encode(&pt.v, a, a.v_cache, pt.box);
  auto kern = a.slopes || !(a.scale > 0.f) || a.softcap > kCapNear ? prefill_tc_kernel<DT, D, PT_ANY>
              : a.softcap > 0.f            ? prefill_tc_kernel<DT, D, PT_CAP>
                                           : prefill_tc_kernel<DT, D, PT_PLAIN>;
  if (const int rc = allow_smem(reinterpret_cast<const void*>(kern), PtCfg<D>::SMEM, "paged_prefill")) return rc;
  if constexpr (PtCfg<D>::TILES == 2) {
    // the warpgroups' shares after setmaxnreg are what the block is launched with: with fewer registers a thread than
    // that it would wait for them for good
    static const int regs = [] {
      int least = 255;
      for (auto k : {prefill_tc_kernel<DT, D, PT_PLAIN>, prefill_tc_kernel<DT, D, PT_CAP>, prefill_tc_kernel<DT, D, PT_ANY>}) {
        cudaFuncAttributes f;
        least = std::min(least, cudaFuncGetAttributes(&f, k) == cudaSuccess ? f.numRegs : 0);
      }
      return least;
    }();
    if (regs * pt_threads(D) < 128 * 64 + 512 * 104) return fail(SMAQ_ERR_UNSUPPORTED, "paged_prefill: built with %d registers a thread", regs);
  }
  const int64_t units = grid_tiles(a.n_rows, a.batch, p.group, D) * a.n_kv_heads;
  pt.splits = splits_for(units, int64_t(a.max_blocks) * a.page_size);
  pt.spin = exact_wait_limit();
  pt.parts = static_cast<float*>(a.workspace);
  if (units * pt.splits * (pt_rows(D) / PJ_ROWS) >= (int64_t(1) << 31)) return fail(SMAQ_ERR_UNSUPPORTED, "paged_prefill: too many rows");
  const size_t need = prefill_tc_workspace(a.n_rows, a.batch, a.n_q_heads, a.n_kv_heads, D, int64_t(a.max_blocks) * a.page_size);
  if (need && (!a.workspace || a.workspace_bytes < need))
    return fail(SMAQ_ERR_WORKSPACE, "paged_prefill: workspace %zu bytes, needs %zu", a.workspace ? a.workspace_bytes : size_t(0), need);
  if (need && reinterpret_cast<uintptr_t>(a.workspace) % 16) return fail(SMAQ_ERR_INVALID, "paged_prefill: workspace must be 16-byte aligned");
  kern<<<unsigned(units * pt.splits), pt_threads(D), PtCfg<D>::SMEM, st>>>(pt);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || pt.splits == 1) return cuda_status(e, "paged_prefill");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(units * (pt_rows(D) / PJ_ROWS)));
  cfg.blockDim = dim3(PJ_THREADS);
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, prefill_join_kernel<DT, D>, pt), "paged_prefill join");
}

}  // namespace

size_t prefill_tc_workspace(int64_t n_rows, int batch, int n_q_heads, int n_kv_heads, int head_dim, int64_t max_tokens) {
  if (n_rows <= 0 || batch < 0 || n_kv_heads <= 0 || n_q_heads < n_kv_heads) return 0;
  const int64_t units = grid_tiles(n_rows, batch, n_q_heads / n_kv_heads, head_dim) * n_kv_heads;
  const int splits = splits_for(units, max_tokens);
  return splits > 1 ? size_t(units) * splits * part_floats(head_dim) * sizeof(float) : 0;
}

bool prefill_tc_eligible(const smaq_paged_args& a) {
  // Walks of one block leave the tensor cores nothing to overlap: up to 128 tokens of table the warp-level kernel
  // takes 16.5 us a call (host included) where this one takes 20; at 256 tokens both take 20, from 512 on this one wins.
  if (int64_t(a.max_blocks) * a.page_size <= PT_N) return false;
  return a.dtype != SMAQ_F32 && (a.head_dim == 64 || a.head_dim == 128 || a.head_dim == 256) && paged_aligned(a);
}

int launch_prefill_tc(const PagedParams& p, cudaStream_t st) {
  const bool bf16 = p.a.dtype == SMAQ_BF16;
  switch (p.a.head_dim) {
    case 64: return bf16 ? launch<BF16, 64>(p, st) : launch<F16, 64>(p, st);
    case 128: return bf16 ? launch<BF16, 128>(p, st) : launch<F16, 128>(p, st);
    default: return bf16 ? launch<BF16, 256>(p, st) : launch<F16, 256>(p, st);
  }
}

}  // namespace smaq

namespace smaq {
int norm_rope_fault(bool& set);  // norm_rope.cu
}

namespace smaq {
// A poll lasts 4 us (the hardware suspends it): a wait gives up after a second.
static std::atomic<uint32_t> g_wait_limit{1u << 18};
uint32_t exact_wait_limit() { return g_wait_limit.load(std::memory_order_relaxed); }
}  // namespace smaq

extern "C" void smaq_exact_set_wait_limit(int64_t polls) {
  smaq::g_wait_limit.store(polls < 0 ? 1u << 18 : uint32_t(std::min<int64_t>(polls, 1 << 18)), std::memory_order_relaxed);
}

extern "C" int smaq_exact_status(void* stream) {
  cudaError_t e = cudaStreamSynchronize(static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return smaq::cuda_status(e, "exact status: stream");
  unsigned int word = 0, zero = 0;
  e = cudaMemcpyFromSymbol(&word, smaq::g_prefill_fault, sizeof(word));
  if (e == cudaSuccess && word) e = cudaMemcpyToSymbol(smaq::g_prefill_fault, &zero, sizeof(zero));
  if (e != cudaSuccess) return smaq::cuda_status(e, "exact status: read");
  bool rope = false;
  if (const int st = smaq::norm_rope_fault(rope)) return st;
  if (word || rope) return smaq::fail(SMAQ_ERR_DEVICE, "%s: a bounded device wait ran out", word ? "paged_prefill" : "norm_rope");
  return SMAQ_OK;
}
