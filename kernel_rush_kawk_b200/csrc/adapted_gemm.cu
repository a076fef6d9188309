// A projection with the low-rank adapters of its rows in one product on the 5th-generation tensor cores:
// C[r, n] = sum_k x[r, k] W[n, k] + sum_j t[r, p of n, j] B[a, n, j], bfloat16 in and out, float32 sums, rounded once. The adapters' second factors
// are further blocks of k: behind W's columns come, for every adapter a that a tile of rows has, B's rows of a beside the rows' t, which are zero
// for rows that have another. Gated: W and B hold gate rows and then up rows, and C = silu(g) u.
//
// first_factor_tiles_kernel makes t = scale (x A^T), rounded to bfloat16 (half a step of 2^-8 of a sum that is itself a part of the result, which is
// rounded the same way), by mma.sync: 16 rows and 16 ranks a block, K dealt to its eight warps.
//
// adapted_gemm_kernel works in pairs of blocks (cta_group::2): 256 rows of W are the product's M, half of them in each block's shared memory, and a
// tile's rows, 32 to 256, its N. So a product costs what it has rows, in steps of 32, and W passes once for up to 256 of them. Pairs stay
// and walk the tiles; an accumulator is half of tensor memory, so that one tile is read back while the next is multiplied.
//   Whole tiles: every pair takes tiles in turn, the row tiles of 256 columns side by side, and writes C.
//   Shares: for few rows, where W's bytes are the cost and there are fewer tiles than pairs. The blocks of k of all tiles are
//   dealt to the pairs in equal runs; what a pair has of a tile goes to scratch in 32 bits, and finish_kernel adds a tile's shares in order.
//
// Warp 0 of either block drives TMA (64 elements of k a stage, 128-byte swizzle) and counts on the first block's barriers; warp 1 of the first
// block issues tcgen05.mma for both; warps 2 to 9 read accumulators back: a lane is a column of C there and what it holds are rows, so a warp turns
// 32 x 32 of them through a patch of shared memory. Gate and up rows alternate in the tile, so that neighbouring lanes hold a column's
// two sums. Every wait is bounded: one that runs out sets the error word, and the blocks leave after freeing their tensor memory.
#include "adapters.cuh"
#include "mma.cuh"
#include "tcgen05.cuh"

namespace {

using namespace tc;

// ---------------------------------------------------------------------------------------------------------------------
// The first factor
// ---------------------------------------------------------------------------------------------------------------------

// t of the row tiles' adapters, [slot of the list][tile_rows][parts * wide]: zeros where a row has another adapter. Blocks of 16 rows (x), of
// the tile's adapters in turn (y), of 16 ranks of a part (z). A warp has every eighth block of 32 k; inside one, lane t's 16 bytes are elements 8 t
// and after for rows and ranks alike, which a sum over k does not mind.
__global__ void __launch_bounds__(256) first_factor_tiles_kernel(bf16* __restrict__ t, const bf16* __restrict__ x, long long ldx, int K, const __grid_constant__ AdapterBank bank,
                                                                 const __grid_constant__ AdapterTiles tiles, int* __restrict__ error) {
  __shared__ float red[8][256];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, q = lane & 3;
  const int r0 = blockIdx.x * 16, tile = r0 / tiles.tile_rows;
  const int chunks = (bank.rank + 15) / 16, part = blockIdx.z / chunks, j0 = blockIdx.z % chunks * 16;
  grid_launch_dependents();
  grid_dependency_wait();
  const int first = tiles.info[2 * tile], count = tiles.info[2 * tile + 1];
  const int mine = lane < 16 && r0 + lane < tiles.rows ? tiles.row_adapter[r0 + lane] : -1;
  const int width = bank.parts * bank.wide;
  for (int i = blockIdx.y; i < count; i += gridDim.y) {
    const int a = tiles.list[first + i];
    if (a >= bank.capacity) {
      if (threadIdx.x == 0) atomicExch(error, KRK_ERROR_ADAPTER);
      continue;
    }
    const int rank = bank.ranks[a * bank.parts + part];
    if (j0 >= rank) continue;
    const unsigned has = __ballot_sync(0xffffffffu, mine == a);
    bf16* to = t + ((size_t)(first + i) * tiles.tile_rows + (r0 - tile * tiles.tile_rows)) * width + part * bank.wide + j0;
    if (has == 0) {  // columns come in steps of 16, rows of a multiple of 32 bytes
      if (threadIdx.x < 32) *reinterpret_cast<uint4*>(to + (size_t)(threadIdx.x >> 1) * width + (threadIdx.x & 1) * 8) = make_uint4(0, 0, 0, 0);
      continue;
    }
    const bf16* x0 = x + (size_t)min(r0 + g, tiles.rows - 1) * ldx + 8 * q;
    const bf16* x1 = x + (size_t)min(r0 + g + 8, tiles.rows - 1) * ldx + 8 * q;
    const bool row0 = has >> g & 1, row1 = has >> (g + 8) & 1, rank0 = j0 + g < rank, rank1 = j0 + 8 + g < rank;
    const bf16* a0 = reinterpret_cast<const bf16*>(bank.a) + ((size_t)a * bank.parts * bank.rank + part * bank.rank + min(j0 + g, rank - 1)) * K + 8 * q;
    const bf16* a1 = reinterpret_cast<const bf16*>(bank.a) + ((size_t)a * bank.parts * bank.rank + part * bank.rank + min(j0 + 8 + g, rank - 1)) * K + 8 * q;
    float acc[2][4] = {};
    constexpr int DEEP = 5;
    for (int c = warp * 32; c < K; c += 8 * 32 * DEEP) {
      uint4 xv[DEEP][2], av[DEEP][2];
#pragma unroll
      for (int d = 0; d < DEEP; ++d) {
        const int k = c + d * 256;
        const bool in = k + 8 * q < K;  // K is a multiple of 8
        const uint4 zero = make_uint4(0, 0, 0, 0);
        av[d][0] = in && rank0 ? ld_stream_16(a0 + k) : zero;
        av[d][1] = in && rank1 ? ld_stream_16(a1 + k) : zero;
        xv[d][0] = in && row0 ? *reinterpret_cast<const uint4*>(x0 + k) : zero;
        xv[d][1] = in && row1 ? *reinterpret_cast<const uint4*>(x1 + k) : zero;
      }
#pragma unroll
      for (int d = 0; d < DEEP; ++d)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          mma_bf16_16816(acc[h], xv[d][0].x, xv[d][1].x, xv[d][0].y, xv[d][1].y, av[d][h].x, av[d][h].y);
          mma_bf16_16816(acc[h], xv[d][0].z, xv[d][1].z, xv[d][0].w, xv[d][1].w, av[d][h].z, av[d][h].w);
        }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int c = 0; c < 4; ++c) red[warp][(g + (c >> 1) * 8) * 16 + h * 8 + 2 * q + (c & 1)] = acc[h][c];
    __syncthreads();
    const int row = threadIdx.x >> 4, j = threadIdx.x & 15;
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) sum += red[w][threadIdx.x];
    const bool live = (has >> row & 1) && j0 + j < rank;
    to[(size_t)row * width + j] = from_float<bf16>(live ? sum * bank.scale[a * bank.parts + part] : 0.f);
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// The product
// ---------------------------------------------------------------------------------------------------------------------

constexpr int BK = 64, UMMA_K = 16;
constexpr int PAIRS = 74;
constexpr int READERS = 8;  // warps that read accumulators: two to a quarter of tensor memory's lanes
constexpr int THREADS = 64 + 32 * READERS;
constexpr uint32_t W_BYTES = 128 * BK * 2;  // a block's half of the pair's weights
constexpr int BUF_COLS = 256;               // tensor memory of an accumulator; there are two
constexpr int PATCH_PITCH = 80;             // bytes of a row of a warp's patch for the transpose: 16-byte reads of 32 rows meet no bank twice
constexpr int PATCH_BYTES = 32 * PATCH_PITCH;
constexpr int RING_BYTES = 196 * 1024, MOST_STAGES = 10;
constexpr size_t SMEM_BYTES = 1024 + (size_t)RING_BYTES + READERS * PATCH_BYTES + (2 * MOST_STAGES + 5) * 8 + (MOST_STAGES + 4) * 4;

struct Maps {
  CUtensorMap x, w, t, b[KRK_MAX_PARTS];
};

__device__ __forceinline__ void tma_load_4d_pair(void* smem_dst, const CUtensorMap* map, uint32_t cluster_bar, int x, int y, int z, int u) {
  asm volatile(
      "cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
      ::"r"(smem_u32(smem_dst)), "l"(map), "r"(cluster_bar), "r"(x), "r"(y), "r"(z), "r"(u)
      : "memory");
}
__device__ __forceinline__ void umma_bf16_pair_warp(uint32_t tmem_d, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n.reg .pred p, q;\n"
      "elect.sync _|q, 0xffffffff;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "@q tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}"
      ::"r"(tmem_d), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_commit_pair_warp(uint64_t* bar) {
  asm volatile(
      "{\n.reg .pred q;\n"
      "elect.sync _|q, 0xffffffff;\n"
      "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n}"
      ::"r"(smem_u32(bar)), "h"((uint16_t)3)
      : "memory");
}

// The work of a pair. Whole tiles: tiles pair, pair + pairs, ... . Shares: of the units of all tiles (a tile's blocks of k, then its adapters, each
// one unit) in order, `run` from pair * run on.
struct Walk {
  int units, run, at, end;  // units a tile; the next unit and the last (shares)
  __device__ Walk(int pair, int units_, int tiles, int pairs) : units(units_) {
    const long long all = (long long)units * tiles;
    run = (int)((all + pairs - 1) / pairs);
    at = (int)min((long long)pair * run, all);
    end = (int)min((long long)at + run, all);
  }
};

template <bool GATED, bool SHARES>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS)
adapted_gemm_kernel(const __grid_constant__ Maps maps, void* __restrict__ out, int N, int K, const __grid_constant__ AdapterBank bank,
                    const __grid_constant__ AdapterTiles tiles, int* __restrict__ error) {
  constexpr int BC = GATED ? 64 : 128;  // columns of C a block makes of a tile; the pair twice as many
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* ring = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  unsigned char* patches = ring + RING_BYTES;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(patches + READERS * PATCH_BYTES);  // the first block's: copies of both have landed
  uint64_t* empty_bar = full_bar + MOST_STAGES;   // either block's: the products have read a stage
  uint64_t* acc_full = empty_bar + MOST_STAGES;   // either block's
  uint64_t* acc_empty = acc_full + 2;             // the first block's: the reading warps of both are through
  uint64_t* drain_bar = acc_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain_bar + 1);
  int* issued = reinterpret_cast<int*>(tmem_slot + 1);  // blocks of k that were asked for, where a wait ran out; else -1
  volatile int* steps = issued + 1;  // [stages] of 16 k in the stage; 256 more: the tile's last
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();

  if (threadIdx.x == 0) {
    for (int s = 0; s < MOST_STAGES; ++s) {
      mbar_init(full_bar + s, 1);
      mbar_init(empty_bar + s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(acc_full + b, 1);
      mbar_init(acc_empty + b, 2 * READERS);
    }
    mbar_init(drain_bar, 1);
    *issued = -1;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(2 * BUF_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // the other block's barriers exist
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  grid_launch_dependents();
  grid_dependency_wait();
  const int half = tiles.tile_rows / 2;  // rows that each block of the pair brings
  const uint32_t stage_bytes = W_BYTES + (uint32_t)half * BK * 2;
  const int stages = min(MOST_STAGES, (int)(RING_BYTES / stage_bytes));
  const int k_blocks = (K + BK - 1) / BK, row_tiles = (tiles.rows + tiles.tile_rows - 1) / tiles.tile_rows;
  const int all_tiles = row_tiles * ((N + 2 * BC - 1) / (2 * BC));
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  Walk walk(pair, k_blocks + (SHARES ? tiles.info[1] : 0), all_tiles, pairs);  // (shares have a single row tile)
  // the tiles of this pair, in order: t, and for shares its units from u0 to u1
  auto next_tile = [&](int& t, int& u0, int& u1) {
    if (SHARES) {
      if (walk.at >= walk.end) return false;
      t = walk.at / walk.units;
      u0 = walk.at - t * walk.units;
      u1 = min(walk.units, u0 + walk.end - walk.at);
      walk.at += u1 - u0;
      return true;
    }
    t = t < 0 ? pair : t + pairs;
    u0 = 0;
    u1 = INT_MAX;
    return t < all_tiles;
  };
  int t = -1, u0, u1;

  if (warp == 0) {
    int s = 0, asked = 0;
    uint32_t parity = 1;  // of the round before: a first round finds its stages empty
    bool ok = true;
    const uint32_t bytes = 2 * stage_bytes;
    // a stage to fill, by one lane
    auto enter = [&](int what) {
      if (!mbar_wait(empty_bar + s, parity)) {
        atomicExch(error, 3);
        *issued = asked;
        return false;
      }
      if (rank == 0) {
        steps[s] = what;
        mbar_expect_tx(full_bar + s, bytes);
      }
      ++asked;
      return true;
    };
    while (ok && next_tile(t, u0, u1)) {
      const int rt = t % row_tiles, wt = t / row_tiles, f0 = (wt * 2 + (int)rank) * BC, m0 = rt * tiles.tile_rows + (int)rank * half;
      const int first = tiles.info[2 * rt], count = tiles.info[2 * rt + 1];
      // which parts the pair's columns reach into (gated: both)
      int p0 = 0, p1 = bank.parts;
      if (!GATED) {
        p0 = part_of(bank, wt * 2 * BC);
        p1 = part_of(bank, min(N, (wt + 1) * 2 * BC) - 1) + 1;
      }
      const int e0 = max(0, u0 - k_blocks), e1 = min(count, u1 - k_blocks);  // adapters of the list
      // a lane's adapter of the list, and its parts' ranks in steps of 16, a byte each
      int a = -1;
      uint32_t ranks = 0;
      auto look = [&](int i) {
        a = i + lane < e1 ? tiles.list[first + i + lane] : -1;
        ranks = 0;
        if (a >= 0 && a < bank.capacity)
          for (int p = p0; p < p1; ++p) ranks |= (uint32_t)((bank.ranks[a * bank.parts + p] + 15) / 16) << 8 * p;
      };
      int left = 0;  // blocks of k that the adapters make
      for (int i = e0; i < e1; i += 32) {
        look(i);
        int n = 0;
        for (int p = p0; p < p1; ++p) n += ((ranks >> 8 * p & 255) + 3) / 4;
        left += __reduce_add_sync(0xffffffffu, n);
      }
      const int k1 = min(k_blocks, u1);
      if (lane == 0) {
        for (int kb = u0; kb < k1 && ok; ++kb) {
          if (!(ok = enter(4 | (kb + 1 == k1 && left == 0 ? 256 : 0)))) break;
          unsigned char* stage = ring + s * stage_bytes;
          const uint32_t bar = cluster_address(full_bar + s, 0);
          if (GATED) tma_load_3d_pair(stage, &maps.w, bar, kb * BK, 0, f0);
          else tma_load_2d_pair(stage, &maps.w, bar, kb * BK, f0);
          tma_load_2d_pair(stage + W_BYTES, &maps.x, bar, kb * BK, m0);
          if (++s == stages) { s = 0; parity ^= 1; }
        }
        if (SHARES && ok && u0 >= k1 && left == 0) {  // a share of adapters that leave these columns as they are: zeros from behind the last k
          if ((ok = enter(1 | 256))) {
            unsigned char* stage = ring + s * stage_bytes;
            const uint32_t bar = cluster_address(full_bar + s, 0);
            if (GATED) tma_load_3d_pair(stage, &maps.w, bar, k_blocks * BK, 0, f0);
            else tma_load_2d_pair(stage, &maps.w, bar, k_blocks * BK, f0);
            tma_load_2d_pair(stage + W_BYTES, &maps.x, bar, k_blocks * BK, m0);
            if (++s == stages) { s = 0; parity ^= 1; }
          }
        }
      }
      for (int i = e0; i < e1; ++i) {
        if ((i - e0) % 32 == 0) look(i);
        const int ai = __shfl_sync(0xffffffffu, a, (i - e0) % 32);
        const uint32_t of = __shfl_sync(0xffffffffu, ranks, (i - e0) % 32);
        if (lane == 0 && ok)
          for (int p = p0; p < p1 && ok; ++p)
            for (int r = of >> 8 * p & 255, kb = 0; r > 0; r -= 4, ++kb) {
              --left;
              if (!(ok = enter(min(r, 4) | (left == 0 ? 256 : 0)))) break;
              unsigned char* stage = ring + s * stage_bytes;
              const uint32_t bar = cluster_address(full_bar + s, 0);
              if (GATED) tma_load_4d_pair(stage, &maps.b[p], bar, kb * BK, -p, f0, ai);
              else tma_load_3d_pair(stage, &maps.b[p], bar, kb * BK, f0 - bank.begin[p], ai);
              tma_load_2d_pair(stage + W_BYTES, &maps.t, bar, p * bank.wide + kb * BK, (first + i) * tiles.tile_rows + (int)rank * half);
              if (++s == stages) { s = 0; parity ^= 1; }
            }
      }
      ok = __shfl_sync(0xffffffffu, ok, 0);
    }
    if (lane == 0 && ok)  // the last stages' releases, too, have arrived before the block leaves
      for (int i = 0; i < stages; ++i) {
        if (!mbar_wait(empty_bar + s, parity)) {
          atomicExch(error, 3);
          *issued = asked;
          break;
        }
        if (++s == stages) { s = 0; parity ^= 1; }
      }
  } else if (warp == 1) {
    int s = 0, buf = 0;
    uint32_t parity = 0, acc_parity = 1;
    bool ok = rank == 0;
    const uint32_t idesc = umma_idesc(256, tiles.tile_rows);
    while (ok && next_tile(t, u0, u1)) {
      const uint32_t acc = tmem_base + (uint32_t)buf * BUF_COLS;
      ok = mbar_wait(acc_empty + buf, acc_parity);  // both blocks have read what was there
      ok = __all_sync(0xffffffffu, ok);
      tc_fence_after();
      uint32_t more = 0;
      for (bool last = false; ok && !last;) {
        ok = __all_sync(0xffffffffu, mbar_wait(full_bar + s, parity));
        if (!ok) break;
        tc_fence_after();
        const int what = steps[s];
        last = what >> 8;
        unsigned char* stage = ring + s * stage_bytes;
        const uint64_t w_desc = umma_desc(stage), r_desc = umma_desc(stage + W_BYTES);
        if ((what & 255) == 4) {
#pragma unroll
          for (int k = 0; k < BK / UMMA_K; ++k) {
            const uint64_t adv = (uint64_t)((k * UMMA_K * 2) >> 4);
            umma_bf16_pair_warp(acc, w_desc + adv, r_desc + adv, idesc, more);
            more = 1;
          }
        } else {
          for (int k = 0; k < (what & 255); ++k) {
            const uint64_t adv = (uint64_t)((k * UMMA_K * 2) >> 4);
            umma_bf16_pair_warp(acc, w_desc + adv, r_desc + adv, idesc, more);
            more = 1;
          }
        }
        umma_commit_pair_warp(empty_bar + s);
        if (++s == stages) { s = 0; parity ^= 1; }
      }
      if (ok) {
        umma_commit_pair_warp(acc_full + buf);
      } else {  // products on their way end before tensor memory is freed
        if (lane == 0) atomicExch(error, 4);
        umma_commit_pair_warp(drain_bar);
        mbar_wait(drain_bar, 0, WAIT_LIMIT_NS / 20);
      }
      buf ^= 1;
      acc_parity ^= buf == 0;
    }
  } else {
    const int quarter = warp & 3;
    unsigned char* patch = patches + (warp - 2) * PATCH_BYTES;
    int buf = 0;
    uint32_t parity = 0;
    while (next_tile(t, u0, u1)) {
      if (!__all_sync(0xffffffffu, mbar_wait(acc_full + buf, parity))) {
        if (lane == 0) atomicExch(error, 5);
        break;
      }
      tc_fence_after();
      const int rt = t % row_tiles, wt = t / row_tiles, m0 = rt * tiles.tile_rows;
      const int live_rows = min(tiles.tile_rows, tiles.rows - m0);
      const uint32_t acc = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)buf * BUF_COLS;
      if (SHARES) {
        // [share of the tile][row][column of W, gate and up in turn where gated]: a lane's column, 32 of them side by side
        const int first_pair = (int)((long long)t * walk.units / walk.run);
        const int column = (wt * 2 + (int)rank) * 128 + quarter * 32 + lane, columns = GATED ? 2 * N : N;
        float* dst = reinterpret_cast<float*>(out) + (size_t)(pair - first_pair) * tiles.rows * columns + column;
        for (int c0 = (warp - 2) / 4 * 32; c0 < live_rows; c0 += 32 * (READERS / 4)) {
          uint32_t v[32];
          tmem_ld_32x32(acc + (uint32_t)c0, v);
          tmem_wait_ld();
          if (column < columns) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (c0 + j < live_rows) dst[(size_t)(c0 + j) * columns] = __uint_as_float(v[j]);
          }
        }
      } else {
        constexpr int MINE = BC / 4;  // columns of this warp
        const int f0 = (wt * 2 + (int)rank) * BC + quarter * MINE;
        if (f0 < N) {
          for (int c0 = (warp - 2) / 4 * 32; c0 < live_rows; c0 += 32 * (READERS / 4)) {
            uint32_t v[32];
            tmem_ld_32x32(acc + (uint32_t)c0, v);
            tmem_wait_ld();
            if constexpr (GATED) {
              // an even lane has a column's gate and the odd one after it the same column's up: they share the rows, the even ones to the even lane
              const bool odd = lane & 1;
#pragma unroll
              for (int j = 0; j < 16; ++j) {
                const float a = __uint_as_float(v[2 * j]), b = __uint_as_float(v[2 * j + 1]);
                const float got = __shfl_xor_sync(0xffffffffu, odd ? a : b, 1);
                const float gate = odd ? got : a, up = odd ? b : got;
                *reinterpret_cast<bf16*>(patch + (2 * j + (odd ? 1 : 0)) * PATCH_PITCH + (lane >> 1) * 2) =
                    from_float<bf16>(__fdividef(gate, 1.0f + __expf(-gate)) * up);
              }
            } else {
#pragma unroll
              for (int j = 0; j < 32; ++j) *reinterpret_cast<bf16*>(patch + j * PATCH_PITCH + lane * 2) = from_float<bf16>(__uint_as_float(v[j]));
            }
            __syncwarp();
            if (c0 + lane < live_rows) {
              bf16* dst = reinterpret_cast<bf16*>(out) + (size_t)(m0 + c0 + lane) * N + f0;
#pragma unroll
              for (int j = 0; j < MINE; j += 8)  // N is a multiple of 8
                if (f0 + j < N) *reinterpret_cast<uint4*>(dst + j) = *reinterpret_cast<const uint4*>(patch + lane * PATCH_PITCH + j * 2);
            }
            __syncwarp();
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(cluster_address(acc_empty + buf, 0));
      buf ^= 1;
      parity ^= buf == 0;
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (rank == 0 && threadIdx.x == 0 && *issued >= 0)  // copies on their way end before shared memory is given up
    for (int i = max(0, *issued - stages); i < *issued; ++i) mbar_wait(full_bar + i % stages, (uint32_t)(i / stages) & 1u, WAIT_LIMIT_NS / 20);
  __syncthreads();
  cluster_sync();  // neither block's barriers are signalled any more
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(2 * BUF_COLS) : "memory");
  }
}

// The shares of a tile's columns, added in the pairs' order. A block has a tile's 256 columns of W and four rows.
template <bool GATED>
__global__ void __launch_bounds__(256) finish_kernel(bf16* __restrict__ out, const float* __restrict__ shares, int rows, int columns, int k_blocks, int pairs,
                                                     const int* __restrict__ info) {
  grid_launch_dependents();
  grid_dependency_wait();
  const Walk walk(0, k_blocks + info[1], gridDim.x, pairs);
  const int tile = blockIdx.x, r = blockIdx.y * 4 + threadIdx.x / 64, column = tile * 256 + threadIdx.x % 64 * 4;
  const int count = (int)((((long long)tile + 1) * walk.units - 1) / walk.run - (long long)tile * walk.units / walk.run) + 1;
  if (r >= rows || column >= columns) return;
  const float* from = shares + (size_t)r * columns + column;
  float4 sum = *reinterpret_cast<const float4*>(from);
  for (int i = 1; i < count; ++i) {
    const float4 more = *reinterpret_cast<const float4*>(from + (size_t)i * rows * columns);
    sum.x += more.x;
    sum.y += more.y;
    sum.z += more.z;
    sum.w += more.w;
  }
  if (GATED) {
    *reinterpret_cast<uint32_t*>(out + (size_t)r * (columns / 2) + column / 2) =
        pack_bf16x2(sum.x / (1.0f + expf(-sum.x)) * sum.y, sum.z / (1.0f + expf(-sum.z)) * sum.w);
  } else {
    *reinterpret_cast<uint2*>(out + (size_t)r * columns + column) = make_uint2(pack_bf16x2(sum.x, sum.y), pack_bf16x2(sum.z, sum.w));
  }
}

int make_map(CUtensorMap* map, const void* base, int dims, const cuuint64_t* size, const cuuint64_t* stride, const cuuint32_t* box) {
  EncodeTiled fn = encode_fn();
  if (!fn) return -6;
  const cuuint32_t elem[4] = {1, 1, 1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, dims, const_cast<void*>(base), size, stride, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : -7;
}

// A part's second factors of every adapter: boxes of 128 outputs from any output on, or, gated, of 64 outputs in every second place of 128 rows,
// zeros in the others (the middle index, of one value, is asked for from 0 or from -1 on).
int make_map_b(CUtensorMap* map, const AdapterBank& bank, int part, int N, bool gated) {
  const cuuint64_t R = bank.rank, outs = bank.begin[part + 1] - bank.begin[part];
  const bf16* base = reinterpret_cast<const bf16*>(bank.b) + (size_t)bank.begin[part] * bank.rank;
  if (gated) {
    const cuuint64_t size[4] = {R, 1, outs, (cuuint64_t)bank.capacity}, stride[3] = {outs * R * 2, R * 2, (cuuint64_t)N * R * 2};
    const cuuint32_t box[4] = {64, 2, 64, 1};
    return make_map(map, base, 4, size, stride, box);
  }
  const cuuint64_t size[3] = {R, outs, (cuuint64_t)bank.capacity}, stride[2] = {R * 2, (cuuint64_t)N * R * 2};
  const cuuint32_t box[3] = {64, 128, 1};
  return make_map(map, base, 3, size, stride, box);
}

template <bool GATED, bool SHARES>
int launch_gemm(const Maps& maps, void* out, int N, int K, const AdapterBank& bank, const AdapterTiles& tiles, int pairs, int* error, cudaStream_t stream) {
  static unsigned long long allowed = 0;
  auto kern = adapted_gemm_kernel<GATED, SHARES>;
  const cudaError_t e = allow_shared(kern, SMEM_BYTES, &allowed);
  if (e != cudaSuccess) return (int)e;
  return (int)launch_pdl(kern, dim3(2 * pairs), dim3(THREADS), SMEM_BYTES, stream, maps, out, N, K, bank, tiles, error);
}

}  // namespace

// out [rows, N] (gated: [rows, N / 2]) bfloat16 from x [rows, K] (row stride ldx) and w [N, K] (row stride ldw), by tiles of tile_rows rows. t: scratch of
// `slots` * tile_rows * parts * wide bfloat16, as many slots as the lists have (tiles and sequences together). shares: float32 scratch of
// (74 / tiles of 256 columns, rounded up, and one more) * rows * N, or null for whole tiles; shares take one row tile. spread: how many of a tile's
// adapters are taken side by side by the first factor.
KRK_API int krk_adapted_gemm(void* out, const void* x, long long ldx, const void* w, long long ldw, int rows, int N, int K, const AdapterBank* bank,
                             const int* row_adapter, const int* info, const int* list, int tile_rows, int slots, void* t, float* shares, int gated, int spread,
                             int* error, cudaStream_t stream) {
  if (rows == 0 || N == 0) return 0;
  const int width = gated ? N / 2 : N;
  if (K < 64 || K % 8 || width % 8 || ldx % 8 || ldw % 8 || tile_rows % 32 || tile_rows < 32 || tile_rows > 256 || (shares && rows > tile_rows) || spread < 1 ||
      (((uintptr_t)x | (uintptr_t)w | (uintptr_t)out | (uintptr_t)bank->a | (uintptr_t)bank->b | (uintptr_t)t | (uintptr_t)shares) & 15))
    return -2;
  const AdapterTiles tiles = {row_adapter, info, list, rows, tile_rows};
  const long long all = (long long)((rows + tile_rows - 1) / tile_rows) * ((N + 255) / 256);
  if (all * (K / 64 + 1 + slots) > 0x7fffffffLL || (long long)slots * tile_rows > 0x7fffffffLL) return -3;
  Maps maps;
  int rc = make_map_bf16(&maps.x, x, rows, K, ldx, tile_rows / 2);
  if (rc) return rc;
  rc = gated ? make_map_bf16_3d(&maps.w, w, K, 2, width, (long long)width * ldw, ldw, 2, 64) : make_map_bf16(&maps.w, w, N, K, ldw, 128);
  if (rc) return rc;
  rc = make_map_bf16(&maps.t, t, (long long)slots * tile_rows, bank->parts * bank->wide, bank->parts * bank->wide, tile_rows / 2);
  for (int p = 0; p < bank->parts && !rc; ++p) rc = make_map_b(&maps.b[p], *bank, p, N, gated);
  if (rc) return rc;
  const dim3 grid((rows + 15) / 16, spread, bank->parts * ((bank->rank + 15) / 16));
  rc = (int)launch_pdl(first_factor_tiles_kernel, grid, dim3(256), 0, stream, (bf16*)t, (const bf16*)x, ldx, K, *bank, tiles, error);
  if (rc) return rc;
  const int k_blocks = (K + BK - 1) / BK;
  if (!shares) {
    const int pairs = all < PAIRS ? (int)all : PAIRS;
    return gated ? launch_gemm<true, false>(maps, out, width, K, *bank, tiles, pairs, error, stream)
                 : launch_gemm<false, false>(maps, out, width, K, *bank, tiles, pairs, error, stream);
  }
  rc = gated ? launch_gemm<true, true>(maps, shares, width, K, *bank, tiles, PAIRS, error, stream)
             : launch_gemm<false, true>(maps, shares, width, K, *bank, tiles, PAIRS, error, stream);
  if (rc) return rc;
  const dim3 blocks((N + 255) / 256, (rows + 3) / 4);
  return gated ? (int)launch_pdl(finish_kernel<true>, blocks, dim3(256), 0, stream, (bf16*)out, (const float*)shares, rows, N, k_blocks, PAIRS, info)
               : (int)launch_pdl(finish_kernel<false>, blocks, dim3(256), 0, stream, (bf16*)out, (const float*)shares, rows, N, k_blocks, PAIRS, info);
}
