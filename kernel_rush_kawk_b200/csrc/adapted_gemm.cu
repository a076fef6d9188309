// A projection with the low-rank adapters of its rows in one product on the 5th-generation tensor cores:
// C[r, n] = sum_k x[r, k] W[n, k] + sum_j t[r, p of n, j] B[a, n, j], bfloat16 in and out, float32 sums, rounded once. The adapters' second factors
// are further blocks of k: behind W's columns come, for every adapter a that a tile of rows has, B's rows of a beside the rows' t, which are zero
// for rows that have another. Gated: W and B hold gate rows and then up rows, and C = silu(g) u.
//
// The first factor's kernel (first_factor.cu) makes t, rounded to bfloat16 (half a step of 2^-8 of a sum that is itself a part of the result, which is
// rounded the same way).
//
// Bound by the tensor cores for many rows and by W's bytes for few. Cold, with the first factor's kernel: 2,001 rows of one prompt, rank 16, 4,096 x 6,144 82 us
// (101 GFLOP, 61 us at the measured peak; the library's product alone 79 at the power limit, this 94), 3,963 rows with gate and up of 2,560 x 19,456
// 272 (239), nine prompts, 2,103 rows, of 9,728 x 2,560 with adapters of rank 64 96 (63). By counters the tensor pipe is busy for 80 to 86 % of the product's cycles; before it
// comes the first factor, 9 to 17 us, which takes all of the SMs' memory there. 64 rows of 2,560 x 6,144: eight adapters 18.4 us, sixty of rank up to 32 26 (41 MB,
// 6.2 us), all of rank 32 33 (84 MB, 12.9 us): an adapter is a stage of the ring whatever its rank, some 600 clocks of its
// producer, whatever it loads (boxes as narrow as the rank, swizzled within 32 or 64 bytes, changed nothing). (Sums left in 32 bits and the second factors by
// mma.sync in a kernel behind, 16 columns of eight rows a warp: 256 rows with 120 adapters gained, 95 -> 67 us, most others lost, 64 rows
// with eight 23.6 -> 28.7, since every eight rows read their adapters' B again.)
//
// adapted_gemm_kernel works in pairs of blocks (cta_group::2): 256 rows of W are the product's M, half of them in each block's shared memory, and a
// tile's rows, 32 to 256, its N. So a product costs what it has rows, in steps of 32, and W passes once for up to 256 of them. Pairs stay
// and walk the tiles; an accumulator is half of tensor memory, so that one tile is read back while the next is multiplied.
//   Whole tiles: every pair takes tiles in turn, the row tiles of 256 columns side by side, and writes C.
//   Shares: the blocks of k of the tiles that make no whole round of the pairs (for few rows, where W's bytes are the cost, of all tiles) are dealt to the
//   pairs in equal runs; what a pair has of a tile goes to scratch in 32 bits, and who brings a tile's last share adds them
//   in order.
//
// Warp 0 of either block drives TMA (64 elements of k a stage, 128-byte swizzle) and counts on the first block's barriers; warp 1 of the first
// block issues tcgen05.mma for both; warps 2 to 9 read accumulators back: a lane is a column of C there and what it holds are rows, so a warp turns
// 32 x 32 of them through a patch of shared memory. Gate and up rows alternate in the tile, so that neighbouring lanes hold a column's
// two sums. Every wait is bounded: one that runs out sets the error word, and the blocks leave after freeing their tensor memory.
#include "adapters.cuh"
#include "mma.cuh"
#include "shares.cuh"
#include "warp_copies.cuh"

namespace {

using namespace tc;

// ---------------------------------------------------------------------------------------------------------------------
// The product
// ---------------------------------------------------------------------------------------------------------------------

constexpr int BK = 64, UMMA_K = 16;
constexpr int READERS = 8;  // warps that read accumulators: two to a quarter of tensor memory's lanes
constexpr int THREADS = 64 + 32 * READERS;
constexpr uint32_t W_BYTES = 128 * BK * 2;  // a block's half of the pair's weights
constexpr int PATCH_PITCH = 36;             // words of two rows in a warp's patch for the transpose
constexpr int PATCH_BYTES = 16 * PATCH_PITCH * 4;
constexpr int MOST_STAGES = 7;
constexpr int RING_BYTES = 104 * 1024, DEEP_RING_BYTES = 192 * 1024;  // beside the smaller an SM has room for a block of the first factor's
constexpr size_t BESIDE_BYTES = 1024 + READERS * PATCH_BYTES + (2 * MOST_STAGES + 8) * 8 + (MOST_STAGES + 6) * 4;

struct Maps {
  CUtensorMap x, w, t, b[KRK_MAX_PARTS];
};

__device__ __forceinline__ void umma_bf16_pair_warp(uint32_t tmem_d, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n.reg .pred p, q;\n"
      "elect.sync _|q, 0xffffffff;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "@q tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}"
      ::"r"(tmem_d), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// A stage's four products and its release at once.
__device__ __forceinline__ void umma_stage_pair_warp(uint32_t tmem_d, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate, uint64_t* release) {
  asm volatile(
      "{\n.reg .pred p, q, t;\n.reg .b64 a1, a2, a3, b1, b2, b3;\n"
      "elect.sync _|q, 0xffffffff;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "setp.eq.b32 t, 0, 0;\n"
      "add.u64 a1, %1, 2;\nadd.u64 a2, %1, 4;\nadd.u64 a3, %1, 6;\n"
      "add.u64 b1, %2, 2;\nadd.u64 b2, %2, 4;\nadd.u64 b3, %2, 6;\n"
      "@q tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n"
      "@q tcgen05.mma.cta_group::2.kind::f16 [%0], a1, b1, %3, t;\n"
      "@q tcgen05.mma.cta_group::2.kind::f16 [%0], a2, b2, %3, t;\n"
      "@q tcgen05.mma.cta_group::2.kind::f16 [%0], a3, b3, %3, t;\n"
      "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%5], %6;\n}"
      ::"r"(tmem_d), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(smem_u32(release)), "h"((uint16_t)3)
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

// The wait for a load of tensor memory, after which what it loaded may be used and not before.
__device__ __forceinline__ void tmem_wait_ld_of(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                 "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}

template <bool GATED>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(512)  // (of 320: 128 registers a thread leave room for a block of the first factor's)
adapted_gemm_kernel(const __grid_constant__ Maps maps, bf16* __restrict__ out, float* __restrict__ shares, int* __restrict__ done, int shared, int most_shares, int aligned, int ring_bytes, int N, int K, const __grid_constant__ AdapterBank bank,
                    const __grid_constant__ AdapterTiles tiles, int* __restrict__ error) {
  constexpr int BC = GATED ? 64 : 128;  // columns of C a block makes of a tile; the pair twice as many
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* ring = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  unsigned char* patches = ring + ring_bytes;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(patches + READERS * PATCH_BYTES);  // the first block's: copies of both have landed
  uint64_t* empty_bar = full_bar + MOST_STAGES;   // either block's: the products have read a stage
  uint64_t* acc_full = empty_bar + MOST_STAGES;   // either block's
  uint64_t* acc_empty = acc_full + 2;             // the first block's: the reading warps of both are through
  uint64_t* drain_bar = acc_empty + 2;
  uint64_t* ready_bar = drain_bar + 1;            // [2] the first block's: the second has its accumulators
  uint64_t* grown_bar = ready_bar + 2;            // either block's: the second accumulator is there
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(grown_bar + 1);  // [2]
  int* issued = reinterpret_cast<int*>(tmem_slot + 2);  // blocks of k that were asked for, where a wait ran out; else -1
  volatile int* last = issued + 1;   // whether this block has brought a tile's last share
  volatile int* steps = issued + 2;  // [stages] of 16 k in the stage; 256 more: the tile's last
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
    mbar_init(ready_bar, 1);
    mbar_init(ready_bar + 1, 1);
    mbar_init(grown_bar, 1);
    *issued = -1;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  cluster_sync();  // the other block's barriers exist
  // Two accumulators of a power of two of columns, no fewer than the tile's rows. With tiles of more than 128 rows they are all of tensor memory, and a block of
  // the first factor's may hold some of it yet: the second one is taken when the first tile's products are on their way. Until then no later kernel's
  // blocks are let in, which might take it and wait for this kernel's end.
  const int buf_cols = tiles.tile_rows <= 32 ? 32 : 1 << (32 - __clz(tiles.tile_rows - 1));
  auto take = [&](int buf) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot + buf)), "r"(buf_cols) : "memory");
    __syncwarp();
    if (buf == 1) {
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
      grid_launch_dependents();
      tc_fence_before();
      if (lane == 0) mbar_arrive(grown_bar);
    }
    if (rank == 1 && lane == 0) mbar_arrive_cluster(cluster_address(ready_bar + buf, 0));
  };
  if (warp == 1) take(0);
  if (warp >= 1) asm volatile("bar.sync 1, %0;" ::"n"(THREADS - 32) : "memory");
  tc_fence_after();
  uint32_t tmem[2] = {warp >= 1 ? tmem_slot[0] : 0, 0};
  const int half = tiles.tile_rows / 2;  // rows that each block of the pair brings
  const uint32_t stage_bytes = W_BYTES + (uint32_t)half * BK * 2;
  const int stages = min(MOST_STAGES, (int)(ring_bytes / stage_bytes));
  const int k_blocks = (K + BK - 1) / BK, row_tiles = (tiles.rows + tiles.tile_rows - 1) / tiles.tile_rows;
  const int all_tiles = row_tiles * ((N + 2 * BC - 1) / (2 * BC));
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const bool extras = row_tiles == 1;
  Walk walk(pair, pairs, all_tiles, shared, k_blocks, extras ? tiles.info[1] : 0, aligned);
  int t, k0, k1, e0, e1;

  if (warp == 0) {
    int s = 0, asked = 0;
    uint32_t parity = 1;  // of the round before: a first round finds its stages empty
    bool ok = true;
    const uint32_t ring_at = smem_u32(ring), steps_at = smem_u32(const_cast<int*>(steps)), own_full = smem_u32(full_bar), first_full = cluster_address(full_bar, 0);
    uint32_t stage;
    PairStage to;
    to.bytes = 2 * stage_bytes;
    to.expects = rank == 0;
    // a stage to fill
    auto enter = [&] {
      if (!__all_sync(0xffffffffu, mbar_wait(empty_bar + s, parity))) {
        if (lane == 0) {
          atomicExch(error, 3);
          *issued = asked;
        }
        return ok = false;
      }
      stage = ring_at + s * stage_bytes;
      to.bar = first_full + 8 * s;
      to.own_bar = own_full + 8 * s;
      to.word_at = steps_at + 4 * s;
      ++asked;
      if (++s == stages) { s = 0; parity ^= 1; }
      return true;
    };
    auto shared_block = [&](int what, int kb, int f0, int m0) {
      if (GATED) stage_3d_2d_warp(to, what, stage, &maps.w, kb * BK, 0, f0, stage + W_BYTES, &maps.x, kb * BK, m0);
      else stage_2d_2d_warp(to, what, stage, &maps.w, kb * BK, f0, stage + W_BYTES, &maps.x, kb * BK, m0);
    };
    bool waited = false;
    while (ok && walk.next(t, k0, k1, e0, e1)) {
      const int rt = t % row_tiles, wt = t / row_tiles, f0 = (wt * 2 + (int)rank) * BC, m0 = rt * tiles.tile_rows + (int)rank * half;
      const int first = tiles.info[2 * rt], count = tiles.info[2 * rt + 1];
      // which parts the pair's columns reach into (gated: both)
      int p0 = 0, p1 = bank.parts;
      if (!GATED) {
        p0 = part_of(bank, wt * 2 * BC);
        p1 = part_of(bank, min(N, (wt + 1) * 2 * BC) - 1) + 1;
      }
      if (!extras) e1 = walk.ends(k0, k1) ? count : 0;
      // a lane's adapter of the list, and its parts' ranks in steps of 16, a byte each
      int a = -1;
      uint32_t ranks = 0;
      auto look = [&](int i) {
        a = i + lane < e1 ? tiles.slots[2 * (first + i + lane)] : -1;
        ranks = 0;
        if (a >= bank.capacity) atomicExch(error, KRK_ERROR_ADAPTER);
        else if (a >= 0)
          for (int p = p0; p < p1; ++p) ranks |= (uint32_t)((bank.ranks[a * bank.parts + p] + 15) / 16) << 8 * p;
      };
      int left = 0;  // blocks of k that the adapters make
      for (int i = e0; i < e1; i += 32) {
        look(i);
        int n = 0;
        for (int p = p0; p < p1; ++p) n += ((ranks >> 8 * p & 255) + 3) / 4;
        left += __reduce_add_sync(0xffffffffu, n);
      }
      for (int kb = k0; kb < k1; ++kb) {
        if (!enter()) break;
        shared_block(4 | (kb + 1 == k1 && left == 0 ? 256 : 0), kb, f0, m0);
      }
      // a share of adapters that leave these columns as they are: zeros from behind the last k
      if (ok && k0 >= k1 && left == 0 && enter()) shared_block(1 | 256, k_blocks, f0, m0);
      for (int i = e0; i < e1 && ok; ++i) {
        if ((i - e0) % 32 == 0) look(i);
        if (!waited) grid_dependency_wait();  // t
        waited = true;
        const int ai = __shfl_sync(0xffffffffu, a, (i - e0) % 32);
        const uint32_t of = __shfl_sync(0xffffffffu, ranks, (i - e0) % 32);
        for (int p = p0; p < p1 && ok; ++p)
          for (int r = of >> 8 * p & 255, kb = 0; r > 0; r -= 4, ++kb) {
            --left;
            if (!enter()) break;
            const int what = min(r, 4) | (left == 0 ? 256 : 0), column = p * bank.wide + kb * BK, row = (first + i) * tiles.tile_rows + (int)rank * half;
            if (GATED) stage_4d_2d_warp(to, what, stage, &maps.b[p], kb * BK, -p, f0, ai, stage + W_BYTES, &maps.t, column, row);
            else stage_3d_2d_warp(to, what, stage, &maps.b[p], kb * BK, f0 - bank.begin[p], ai, stage + W_BYTES, &maps.t, column, row);
          }
      }
    }
    if (ok)  // the last stages' releases, too, have arrived before the block leaves
      for (int i = 0; i < stages; ++i) {
        if (!__all_sync(0xffffffffu, mbar_wait(empty_bar + s, parity))) {
          if (lane == 0) {
            atomicExch(error, 3);
            *issued = asked;
          }
          break;
        }
        if (++s == stages) { s = 0; parity ^= 1; }
      }
  } else if (warp == 1) {
    int s = 0, buf = 0;
    uint32_t parity = 0, acc_parity = 1;
    bool ok = rank == 0 && __all_sync(0xffffffffu, mbar_wait(ready_bar, 0));
    if (rank == 0 && !ok && lane == 0) atomicExch(error, 4);
    bool grown = false;
    auto grow = [&] {
      if (grown) return;
      grown = true;
      take(1);
      tmem[1] = tmem_slot[1];
      if (rank == 0 && !__all_sync(0xffffffffu, mbar_wait(ready_bar + 1, 0))) {
        ok = false;
        if (lane == 0) atomicExch(error, 4);
      }
    };
    if (buf_cols <= 128) grow();
    const uint32_t idesc = umma_idesc(256, tiles.tile_rows);
    while (ok && walk.next(t, k0, k1, e0, e1)) {
      if (buf == 1) grow();
      if (!ok) break;
      const uint32_t acc = buf ? tmem[1] : tmem[0];
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
          umma_stage_pair_warp(acc, w_desc, r_desc, idesc, more, empty_bar + s);
        } else {
          for (int k = 0; k < (what & 255); ++k) {
            const uint64_t adv = (uint64_t)((k * UMMA_K * 2) >> 4);
            umma_bf16_pair_warp(acc, w_desc + adv, r_desc + adv, idesc, more || k > 0);
          }
          umma_commit_pair_warp(empty_bar + s);
        }
        more = 1;
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
    grow();
  } else {
    const int quarter = warp & 3;
    unsigned char* patch = patches + (warp - 2) * PATCH_BYTES;
    int buf = 0;
    uint32_t parity = 0;
    while (walk.next(t, k0, k1, e0, e1)) {
      if (!__all_sync(0xffffffffu, mbar_wait_long(acc_full + buf, parity))) {
        if (lane == 0) atomicExch(error, 5);
        break;
      }
      tc_fence_after();
      const int rt = t % row_tiles, wt = t / row_tiles, m0 = rt * tiles.tile_rows;
      const int live_rows = min(tiles.tile_rows, tiles.rows - m0);
      if (buf == 1 && tmem[1] == 0) {  // (the first accumulator is not at 0 where the second is: asked again, to no harm)
        if (!__all_sync(0xffffffffu, mbar_wait(grown_bar, 0))) {
          if (lane == 0) atomicExch(error, 5);
          break;
        }
        tmem[1] = *reinterpret_cast<volatile uint32_t*>(tmem_slot + 1);
        tc_fence_after();
      }
      const uint32_t acc = (buf ? tmem[1] : tmem[0]) + ((uint32_t)(quarter * 32) << 16);
      const int c_first = (warp - 2) / 4 * 32;
      constexpr int C_STEP = 32 * (READERS / 4);
      const int parts = t >= shared ? walk.count(t) : 1;
      // 32 columns of tensor memory at a time, the next ones on their way
      uint32_t v[2][32];
      auto each = [&](auto use) {
        if (c_first < live_rows) tmem_ld_32x32(acc + (uint32_t)c_first, v[0]);
        for (int c0 = c_first; c0 < live_rows; c0 += 2 * C_STEP)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int c = c0 + h * C_STEP;
            if (c >= live_rows) break;
            tmem_wait_ld_of(v[h]);
            if (c + C_STEP < live_rows) tmem_ld_32x32(acc + (uint32_t)(c + C_STEP), v[h ^ 1]);
            use(c, v[h]);
          }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(cluster_address(acc_empty + buf, 0));
      };
      if (parts > 1) {
        // [tile][share][row][256 rows of W, gate and up in turn where gated]: a lane's column, 32 of them side by side
        const size_t share = (size_t)tiles.tile_rows * 256;
        float* mine = shares + (size_t)(t - shared) * most_shares * share + rank * 128;
        float* dst = mine + (pair - walk.first_pair(t)) * share + quarter * 32 + lane;
        each([&](int c, const uint32_t (&w)[32]) {
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (c + j < live_rows) dst[(size_t)(c + j) * 256] = __uint_as_float(w[j]);
        });
        // The block that brings a tile's last share adds them all, in the pairs' order. (The first factor's kernel has set the counts to zero.)
        grid_dependency_wait();
        __threadfence();
        asm volatile("bar.sync 2, %0;" ::"n"(32 * READERS) : "memory");
        if (threadIdx.x == 64) *last = atomicAdd(done + (t - shared) * 2 + rank, 1) == parts - 1;
        asm volatile("bar.sync 2, %0;" ::"n"(32 * READERS) : "memory");
        if (*last) {
          __threadfence();
          constexpr int ROWS = 4, DEEP = 3;  // of the shares of so many rows at once, for a warp
          const int column = lane * 4, n = GATED ? (wt * 2 + (int)rank) * BC + column / 2 : (wt * 2 + (int)rank) * BC + column;
          for (int r0 = (warp - 2) * ROWS; r0 < live_rows; r0 += READERS * ROWS) {
            float4 sum[ROWS];
#pragma unroll
            for (int i = 0; i < ROWS; ++i) sum[i] = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int p = 0; p < parts; p += DEEP) {
              float4 more[DEEP][ROWS];
              // (a row or share too many is read again from the last one, and not added)
#pragma unroll
              for (int d = 0; d < DEEP; ++d)
#pragma unroll
                for (int i = 0; i < ROWS; ++i)
                  more[d][i] = __ldcg(reinterpret_cast<const float4*>(mine + min(p + d, parts - 1) * share + (size_t)min(r0 + i, live_rows - 1) * 256 + column));
#pragma unroll
              for (int d = 0; d < DEEP; ++d)
                if (p + d < parts)
#pragma unroll
                  for (int i = 0; i < ROWS; ++i) {
                    sum[i].x += more[d][i].x;
                    sum[i].y += more[d][i].y;
                    sum[i].z += more[d][i].z;
                    sum[i].w += more[d][i].w;
                  }
            }
#pragma unroll
            for (int i = 0; i < ROWS; ++i)
              if (r0 + i < live_rows && n < N) {  // N is a multiple of 8
                bf16* to = out + (size_t)(m0 + r0 + i) * N + n;
                const float4 s = sum[i];
                if (GATED) *reinterpret_cast<uint32_t*>(to) = pack_bf16x2(s.x / (1.0f + expf(-s.x)) * s.y, s.z / (1.0f + expf(-s.z)) * s.w);
                else *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf16x2(s.x, s.y), pack_bf16x2(s.z, s.w));
              }
          }
        }
      } else {
        constexpr int MINE = BC / 4;  // columns of this warp
        const int f0 = (wt * 2 + (int)rank) * BC + quarter * MINE;
        uint32_t* words = reinterpret_cast<uint32_t*>(patch);
        each([&](int c, const uint32_t (&w)[32]) {
          // The patch has a word for two rows of a column.
          if constexpr (GATED) {
            // an even lane has a column's gate and the odd one after it the same column's up: they share the rows, the even lane takes the first two of four
            const bool odd = lane & 1;
#pragma unroll
            for (int j = 0; j < 32; j += 4) {
              float z[2];
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const float a = __uint_as_float(w[j + i]), b = __uint_as_float(w[j + 2 + i]);
                const float got = __shfl_xor_sync(0xffffffffu, odd ? a : b, 1);
                const float gate = odd ? got : a, up = odd ? b : got;
                // By the fast exponential and quotient, good to 2^-17 (of gates below -87, whose products are below 2^-119 of up, nothing is left); half a step of the
                // result is 2^-8. By expf and a division, which shares have the time for: 3,963 rows of 2,560 x 19,456 278.6 -> 282.6 us cold, 512 rows 61.5 -> 64, 200
                // rows 47 -> 53, 4,000 rows of 320 x 8,192 53 -> 73.
                z[i] = __fdividef(gate, 1.0f + __expf(-gate)) * up;
              }
              words[(j / 2 + (odd ? 1 : 0)) * PATCH_PITCH + (lane >> 1)] = pack_bf16x2(z[0], z[1]);
            }
          } else {
#pragma unroll
            for (int j = 0; j < 32; j += 2) words[j / 2 * PATCH_PITCH + lane] = pack_bf16x2(__uint_as_float(w[j]), __uint_as_float(w[j + 1]));
          }
          __syncwarp();
          // neighbouring lanes take eight columns of two rows each: whole sectors at once (N is a multiple of 8)
          constexpr int PER = MINE / 8, STEP = 32 / PER;
          const int j = lane % PER * 8;
          if (f0 + j < N)
#pragma unroll
            for (int r = lane / PER; r < 16; r += STEP) {
              const uint4 lo = *reinterpret_cast<const uint4*>(words + r * PATCH_PITCH + j), hi = *reinterpret_cast<const uint4*>(words + r * PATCH_PITCH + j + 4);
              bf16* to = out + (size_t)(m0 + c + 2 * r) * N + f0 + j;
              if (c + 2 * r < live_rows)
                *reinterpret_cast<uint4*>(to) = make_uint4(__byte_perm(lo.x, lo.y, 0x5410), __byte_perm(lo.z, lo.w, 0x5410), __byte_perm(hi.x, hi.y, 0x5410),
                                                           __byte_perm(hi.z, hi.w, 0x5410));
              if (c + 2 * r + 1 < live_rows)
                *reinterpret_cast<uint4*>(to + N) = make_uint4(__byte_perm(lo.x, lo.y, 0x7632), __byte_perm(lo.z, lo.w, 0x7632), __byte_perm(hi.x, hi.y, 0x7632),
                                                               __byte_perm(hi.z, hi.w, 0x7632));
            }
          __syncwarp();
        });
      }
      buf ^= 1;
      parity ^= buf == 0;
    }
  }
  __syncwarp();
  grid_dependency_wait();  // who waits for this kernel waits for the first factor's as well
  tc_fence_before();
  __syncthreads();
  if (rank == 0 && threadIdx.x == 0 && *issued >= 0)  // copies on their way end before shared memory is given up
    for (int i = max(0, *issued - stages); i < *issued; ++i) mbar_wait(full_bar + i % stages, (uint32_t)(i / stages) & 1u, WAIT_LIMIT_NS / 20);
  __syncthreads();
  cluster_sync();  // neither block's barriers are signalled any more
  if (warp == 1) {
    tc_fence_after();
    for (int b = 0; b < 2; ++b) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem[b]), "r"(buf_cols) : "memory");
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

template <bool GATED>
int launch_gemm(const Maps& maps, bf16* out, float* shares, int* done, int shared, int most_shares, int aligned, int N, int K, const AdapterBank& bank, const AdapterTiles& tiles,
                int pairs, int* error, cudaStream_t stream) {
  static unsigned long long allowed = 0;
  auto kern = adapted_gemm_kernel<GATED>;
  const cudaError_t e = allow_shared(kern, BESIDE_BYTES + DEEP_RING_BYTES, &allowed);
  if (e != cudaSuccess) return (int)e;
  // tiles of many rows want stages ahead: a block of k of 256 rows takes 650 clocks with four, 590 with five, 575 with six, its products alone 512
  const int ring = tiles.tile_rows <= 128 ? RING_BYTES : DEEP_RING_BYTES;
  return (int)launch_pdl(kern, dim3(2 * pairs), dim3(THREADS), BESIDE_BYTES + ring, stream, maps, out, shares, done, shared, most_shares, aligned, ring, N, K, bank,
                         tiles, error);
}

}  // namespace

// out [rows, N] (gated: [rows, N / 2]) bfloat16 from x [rows, K] (row stride ldx) and w [N, K] (row stride ldw), by tiles of tile_rows rows and 256 rows of w, the
// first `shared` of them as whole ones (a multiple of 74, or all). t: scratch of n_slots * tile_rows * parts * wide bfloat16. shares: float32 scratch of the
// other tiles' number times (74 / their number, rounded up, and one more) * tile_rows * 256, and two words a tile behind that, or null where there are none.
KRK_API int krk_adapted_gemm(void* out, const void* x, long long ldx, const void* w, long long ldw, int rows, int N, int K, const AdapterBank* bank,
                             const int* row_adapter, const int* info, const int* slots, int n_slots, int tile_rows, void* t, float* shares, int shared, int gated,
                             int* error, cudaStream_t stream) {
  if (rows == 0 || N == 0) return 0;
  const int width = gated ? N / 2 : N;
  if (K < 64 || K % 8 || width % 8 || ldx % 8 || ldw % 8 || tile_rows % 32 || tile_rows < 32 || tile_rows > 256 || n_slots < 1 ||
      (((uintptr_t)x | (uintptr_t)w | (uintptr_t)out | (uintptr_t)bank->a | (uintptr_t)bank->b | (uintptr_t)t | (uintptr_t)shares) & 15))
    return -2;
  const AdapterTiles tiles = {row_adapter, info, slots, rows, tile_rows, n_slots};
  const int k_blocks = (K + BK - 1) / BK, row_tiles = (rows + tile_rows - 1) / tile_rows;
  const long long all = (long long)row_tiles * ((N + 255) / 256);
  if (all * (k_blocks + (row_tiles == 1 ? n_slots : 0)) > 0x7fffffffLL || (long long)n_slots * tile_rows > 0x7fffffffLL)  // (adapters are dealt out of a single row tile alone)
    return -3;
  if (shared < 0 || shared > all || (shared < all && (shared % PAIRS || !shares))) return -2;
  Maps maps;
  int rc = make_map_bf16(&maps.x, x, rows, K, ldx, tile_rows / 2);
  if (rc) return rc;
  rc = gated ? make_map_bf16_3d(&maps.w, w, K, 2, width, (long long)width * ldw, ldw, 2, 64) : make_map_bf16(&maps.w, w, N, K, ldw, 128);
  if (!rc) rc = make_map_bf16(&maps.t, t, (long long)n_slots * tile_rows, bank->parts * bank->wide, bank->parts * bank->wide, tile_rows / 2);
  for (int p = 0; p < bank->parts && !rc; ++p) rc = make_map_b(&maps.b[p], *bank, p, N, gated);
  const int rest = (int)(all - shared), most_shares = rest ? shares_of_a_tile(rest) : 0;
  int* done = rest ? reinterpret_cast<int*>(shares + (size_t)rest * most_shares * tile_rows * 256) : nullptr;
  if (!rc) rc = krk_first_factor(t, false, done, 2 * rest, x, ldx, K, *bank, tiles, error, stream);
  if (rc) return rc;
  const int pairs = rest || all > PAIRS ? PAIRS : (int)all;
  const int aligned = rest ? aligned_parts(rest, k_blocks) : 0;
  return gated ? launch_gemm<true>(maps, (bf16*)out, shares, done, shared, most_shares, aligned, width, K, *bank, tiles, pairs, error, stream)
               : launch_gemm<false>(maps, (bf16*)out, shares, done, shared, most_shares, aligned, width, K, *bank, tiles, pairs, error, stream);
}
