#include <cooperative_groups.h>

#include "adapters.cuh"
#include "mma.cuh"
#include "warp_copies.cuh"

namespace {

using namespace tc;

// The four products of a block of 64 k, and its place's release, by a whole warp.
__device__ __forceinline__ void umma_stage_warp(uint32_t tmem_d, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate, uint64_t* release) {
  asm volatile(
      "{\n.reg .pred p, q, t;\n.reg .b64 a1, a2, a3, b1, b2, b3;\n"
      "elect.sync _|q, 0xffffffff;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "setp.eq.b32 t, 0, 0;\n"
      "add.u64 a1, %1, 2;\nadd.u64 a2, %1, 4;\nadd.u64 a3, %1, 6;\n"
      "add.u64 b1, %2, 2;\nadd.u64 b2, %2, 4;\nadd.u64 b3, %2, 6;\n"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a1, b1, %3, t;\n"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a2, b2, %3, t;\n"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a3, b3, %3, t;\n"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%5];\n}"
      ::"r"(tmem_d), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(smem_u32(release))
      : "memory");
}

// The slot of block `index` of n, and what it holds. Of a single tile there are as many blocks as the bank has adapters, which may be fewer than slots. Where the tile
// has more adapters than that, some are none of the bank's and may stand before those that are: the blocks take the latter, in order.
__device__ __forceinline__ int2 take_slot(const AdapterTiles& tiles, int capacity, int index, int n, int& slot) {
  const int2* slots = reinterpret_cast<const int2*>(tiles.slots);
  const int count = tiles.info[1];
  slot = index;
  int2 is = slots[index];
  if (count > n) {
    is.x = -1;
    for (int s = 0; s < count; ++s) {
      const int2 other = slots[s];
      if ((unsigned)other.x < (unsigned)capacity && index-- == 0) {
        slot = s;
        is = other;
        break;
      }
    }
  }
  return is;
}

// The first factor of many requests' adapters, t = scale (x A^T), sums in 32 bits on the tensor cores, rounded to bfloat16 (half a step of 2^-8 of a sum that is itself
// a part of the result, which is rounded the same way). t is of every slot,
// [slot][tile_rows][parts * wide], zeros where a row has another adapter than the slot's.
//
// A cluster has 128 rows of a slot's tile (y) and 64 or 128 of the adapter's ranks, all parts' side by side (z), and its `ways` blocks share k. A block multiplies
// its part of k on the tensor cores, fed by TMA in blocks of 64; it sends its sums of every block's share of the rows to that block's shared memory, in 32
// bits, which adds them in the blocks' order and writes its rows. So a sum's order depends on sizes and on the number of slots alone.
//
// What it costs. It has to read x and the used adapters' A: 2,001 rows of 4,096 are 16 MB, 2.5 us. One cold call of that, rank 16 of three parts, 108
// blocks: 17,700 clocks (9 us) of which the blocks of k take 4,400, 400 each; before them come the wait, tensor memory, the slot and its rows' adapters (4,300) and the
// first copies' way (3,000 with the products behind it), after them the sums' way to their block (2,300), the clusters' meeting (1,700) and the writing (1,800). Long
// runs of k (9,728, 75 blocks): 343 clocks a block of k of four products, a stage's way round and not its bytes: neither copies of only the groups
// of 32 rows that have the adapter (two a block of k: 125 -> 128 us of 2,268 rows with the product; one of 32 or 64 rows: no difference) nor eight places for five
// changed it; places and parities counted instead of divided, and a block's four products asked for at once, took 2,400 rows of 60 requests from 152 to 137 us.
// By single lanes a block of k took 700 clocks.
//
// The product's blocks come in while these run, once what came before is over, and wait for t where they need it; so a ring of few blocks of k is no
// larger than fits beside theirs.
constexpr int FIRST_RANKS = 128, FIRST_STAGES = 8, FIRST_THREADS = 192;
constexpr int FIRST_BYTES = 96 * 1024, FIRST_DEEP_BYTES = 160 * 1024;  // of shared memory, beside the product's blocks and alone

__global__ void __launch_bounds__(FIRST_THREADS, 5)  // (of three that an SM's memory takes: in 64 registers they fit beside the product's)
first_factor_tiles_kernel(bf16* __restrict__ t, int* __restrict__ done, int n_done, const __grid_constant__ CUtensorMap map_x,
                                                                           const __grid_constant__ CUtensorMap map_a, int K,
                                                                           const __grid_constant__ AdapterBank bank, const __grid_constant__ AdapterTiles tiles,
                                                                           int ways, int stages, int ring_bytes, int box_rows, int box_ranks, int* __restrict__ error) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* ring = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  // [ways][this block's rows][pitch]; of a block by itself, in the ring's place when that has done its work
  float* inbox = reinterpret_cast<float*>(ways > 1 ? ring + ring_bytes : ring);
  const int pitch = box_ranks + 4;
  __shared__ uint64_t full_bar[FIRST_STAGES], empty_bar[FIRST_STAGES], acc_bar;
  __shared__ uint32_t tmem_slot;
  __shared__ int asked_for;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, way = blockIdx.x % ways;
  if (ways > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // "I have started"
  grid_dependency_wait();
  // Tensor memory is taken before the product's blocks are let in, which take what is left and wait for what these make. They are let in here, since
  // they read what earlier kernels wrote before they wait.
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(FIRST_RANKS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  grid_launch_dependents();
  const uint32_t acc = tmem_slot;
  if (ways > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // every block of the cluster has started
  auto leave = [&] {
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(acc), "r"(FIRST_RANKS) : "memory");
  };
  if (blockIdx.x + blockIdx.y + blockIdx.z == 0)
    for (int i = threadIdx.x; i < n_done; i += FIRST_THREADS) done[i] = 0;  // the product's counts of shares
  int slot;
  const int2 is = take_slot(tiles, bank.capacity, blockIdx.x / ways, gridDim.x / ways, slot);
  const int a = is.x, r0 = is.y * tiles.tile_rows + blockIdx.y * 128;
  if (a < 0 || a >= bank.capacity) return leave();  // the whole cluster (the product says so)
  const int here = min(128, min(tiles.tile_rows - (int)blockIdx.y * 128, tiles.rows - r0));  // rows
  if (here <= 0) return leave();
  namespace cg = cooperative_groups;
  const int share = (here + ways - 1) / ways;  // of the rows
  bool has = false;
  for (int r = threadIdx.x; r < here; r += FIRST_THREADS) has |= tiles.row_adapter[r0 + r] == a;
  const int k_blocks = (K + 63) / 64, each = (k_blocks + ways - 1) / ways, b0 = min(way * each, k_blocks), b1 = min(b0 + each, k_blocks);
  const int n0 = blockIdx.z * box_ranks, per_adapter = bank.parts * bank.rank;
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(full_bar + s, 1);
      mbar_init(empty_bar + s, 1);
    }
    mbar_init(&acc_bar, 1);
    asked_for = -1;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  has = __syncthreads_or(has);
  if (has) {  // the same for the whole cluster
    const uint32_t bytes = (uint32_t)(box_rows + box_ranks) * 128;
    if (warp == 0) {
      int s = 0;
      uint32_t parity = 1;  // (the first round's places are free)
      for (int b = b0; b < b1; ++b) {
        if (!__all_sync(0xffffffffu, mbar_wait(empty_bar + s, parity))) {
          if (lane == 0) {
            atomicExch(error, 3);
            asked_for = b - b0;
          }
          break;
        }
        const uint32_t stage = smem_u32(ring) + s * bytes, bar = smem_u32(full_bar + s);
        two_loads_warp(stage, &map_x, b * 64, r0, stage + box_rows * 128, &map_a, b * 64, a * per_adapter + n0, bar, bytes);
        if (++s == stages) {
          s = 0;
          parity ^= 1;
        }
      }
    } else if (warp == 1) {
      const uint32_t idesc = umma_idesc(128, box_ranks);  // (rows beyond the copies' give rows that nobody reads)
      const uint64_t x_desc = umma_desc(ring), a_desc = umma_desc(ring + box_rows * 128);
      int s = 0;
      uint32_t parity = 0;
      for (int b = b0; b < b1; ++b) {
        if (!__all_sync(0xffffffffu, mbar_wait(full_bar + s, parity))) {
          if (lane == 0) atomicExch(error, 4);
          break;
        }
        tc_fence_after();
        const uint64_t at = s * (bytes >> 4);
        umma_stage_warp(acc, x_desc + at, a_desc + at, idesc, b > b0, empty_bar + s);
        if (++s == stages) {
          s = 0;
          parity ^= 1;
        }
      }
      umma_commit_warp(&acc_bar);  // arrives even after a failed wait, so that all move on
    }
    if (!__all_sync(0xffffffffu, mbar_wait(&acc_bar, 0)) && lane == 0) atomicExch(error, 5);
    __syncthreads();
    if (threadIdx.x == 0 && asked_for >= 0)  // copies on their way end before their place is given up
      for (int i = max(0, asked_for - stages); i < asked_for; ++i) mbar_wait(full_bar + i % stages, (uint32_t)(i / stages) & 1u, WAIT_LIMIT_NS / 20);
    __syncthreads();
    if (warp >= 2 && (warp & 3) * 32 < here) {
      const int row = (warp & 3) * 32 + lane;
      float* to = (ways > 1 ? cg::this_cluster().map_shared_rank(inbox, row < here ? row / share : 0) : inbox) + (way * share + row % share) * pitch;
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < FIRST_RANKS; c += 32) {
        if (c >= box_ranks) break;
        uint32_t v[32];
        tmem_ld_32x32(acc + ((uint32_t)((warp & 3) * 32) << 16) + c, v);
        tmem_wait_ld();
        if (row < here)
#pragma unroll
          for (int j = 0; j < 32; j += 4)
            if (c + j < box_ranks)
              *reinterpret_cast<float4*>(to + c + j) =
                  b1 > b0 ? make_float4(__uint_as_float(v[j]), __uint_as_float(v[j + 1]), __uint_as_float(v[j + 2]), __uint_as_float(v[j + 3])) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
      tc_fence_before();
    }
    __syncthreads();
    tc_fence_after();
  }
  leave();  // (nobody who holds tensor memory waits for another block's end)
  if (has && ways > 1) cluster_sync();
  // eight ranks of a row a thread
  const int first_row = way * share, rows = min(share, here - first_row), groups = box_ranks / 8;
  const int width = bank.parts * bank.wide;
  for (int o = threadIdx.x; o < rows * groups; o += FIRST_THREADS) {
    const int mine = o / groups, row = first_row + mine, c = o % groups * 8, part = (n0 + c) / bank.rank, j = (n0 + c) % bank.rank;
    if (part >= bank.parts) continue;
    uint4 pack = make_uint4(0, 0, 0, 0);
    if (tiles.row_adapter[r0 + row] == a) {
      const int rank = bank.ranks[a * bank.parts + part];
      const float scale = bank.scale[a * bank.parts + part];
      float v[8] = {};
      for (int w = 0; w < ways; ++w) {
        const float* from = inbox + (w * share + mine) * pitch + c;
        const float4 lo = *reinterpret_cast<const float4*>(from), hi = *reinterpret_cast<const float4*>(from + 4);
        v[0] += lo.x; v[1] += lo.y; v[2] += lo.z; v[3] += lo.w;
        v[4] += hi.x; v[5] += hi.y; v[6] += hi.z; v[7] += hi.w;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = j + i < rank ? v[i] * scale : 0.f;
      pack = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
    }
    bf16* to = t + ((size_t)slot * tiles.tile_rows + blockIdx.y * 128 + row) * width + part * bank.wide + j;
    *reinterpret_cast<uint4*>(to) = pack;
    if (j + 8 == bank.rank && bank.wide > bank.rank) *reinterpret_cast<uint4*>(to + 8) = make_uint4(0, 0, 0, 0);  // the product takes whole steps of sixteen
  }
}

// The same for adapters that few rows have each, of one tile: memory is what bounds it, and neither tensor memory nor clusters are worth their way. A block has 16 of a
// slot's ranks and all of k, a warp a part of it, five blocks of 32 k on their way to registers at a time; the ranks are a product's M, up to 16 of the
// adapter's rows, wherever they are, its N. The warps' sums are added in order: a sum's order depends on K alone.
//
// COMPACT: t of every row, for up to 16 rows (the tiles' form served these before: 16 rows with nine adapters of rank 16, the product with it, cold, 9,728 x 2,560 24.6 us
// and 20.5 here, 4,096 x 2,560 18.4 and 16.4; one row of 2,560 x 6,144 14.3 and 12.3 to 14.4, the timer's steps being 2; sixteen adapters of rank 64 beside 4,096 x 24,576 61 and 65). By eight
// warps a long k takes more rounds of loads: one row of 9,728 x 2,560 22.5, by sixteen 18.4.
constexpr int FEW_DEEP = 5, FEW_RANKS = 16;

template <bool COMPACT, int WARPS>
__global__ void __launch_bounds__(32 * WARPS, 16 / WARPS)
first_factor_few_kernel(bf16* __restrict__ t, int* __restrict__ done, int n_done, const bf16* __restrict__ x, long long ldx, int K, const __grid_constant__ AdapterBank bank,
                        const __grid_constant__ AdapterTiles tiles) {
  __shared__ float sums[WARPS][FEW_RANKS][17];
  __shared__ int list[256], listed;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, q = lane & 3;
  grid_dependency_wait();
  grid_launch_dependents();
  if (blockIdx.x + blockIdx.y == 0)
    for (int i = tid; i < n_done; i += 32 * WARPS) done[i] = 0;
  int slot;
  const int a = take_slot(tiles, bank.capacity, blockIdx.y, gridDim.y, slot).x, rows = min(tiles.rows, tiles.tile_rows);
  if (a < 0 || a >= bank.capacity) return;  // (the product says so)
  if (warp == 0) {
    int n = 0;
    for (int r = lane; r - lane < rows; r += 32) {
      const bool has = r < rows && tiles.row_adapter[r] == a;
      const unsigned all = __ballot_sync(0xffffffffu, has);
      if (has) list[n + __popc(all & ((1u << lane) - 1))] = r;
      n += __popc(all);
    }
    if (lane == 0) listed = n;
  }
  __syncthreads();
  const int n = listed, i0 = blockIdx.x * FEW_RANKS, per = bank.parts * bank.rank, width = bank.parts * bank.wide;
  const bf16* w = reinterpret_cast<const bf16*>(bank.a) + ((size_t)a * per + i0 + g) * K + 8 * q;
  const bool w0_there = i0 + g < per, w1_there = i0 + g + 8 < per;
  const int chunks = (K + 31) / 32, each = (chunks + WARPS - 1) / WARPS, c1 = min(chunks, (warp + 1) * each);
  const uint4 zero = make_uint4(0, 0, 0, 0);
  bf16* to = t + (COMPACT ? 0 : (size_t)slot * tiles.tile_rows * width);
  for (int m0 = 0; m0 < n; m0 += 16) {
    const int row[2] = {m0 + g < n ? list[m0 + g] : -1, m0 + 8 + g < n ? list[m0 + 8 + g] : -1};
    const bf16* from[2] = {x + max(row[0], 0) * ldx + 8 * q, x + max(row[1], 0) * ldx + 8 * q};
    float acc[2][4] = {};
    for (int c = warp * each; c < c1; c += FEW_DEEP) {
      uint4 w4[FEW_DEEP][2], x4[FEW_DEEP][2];
#pragma unroll
      for (int d = 0; d < FEW_DEEP; ++d) {
        const int k = (c + d) * 32;
        const bool in = c + d < c1 && k + 8 * q < K;
        w4[d][0] = in && w0_there ? ld_stream_16(w + k) : zero;
        w4[d][1] = in && w1_there ? ld_stream_16(w + (size_t)8 * K + k) : zero;
#pragma unroll
        for (int h = 0; h < 2; ++h) x4[d][h] = in && row[h] >= 0 ? __ldcg(reinterpret_cast<const uint4*>(from[h] + k)) : zero;
      }
#pragma unroll
      for (int d = 0; d < FEW_DEEP; ++d)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          mma_bf16_16816(acc[h], w4[d][0].x, w4[d][1].x, w4[d][0].y, w4[d][1].y, x4[d][h].x, x4[d][h].y);
          mma_bf16_16816(acc[h], w4[d][0].z, w4[d][1].z, w4[d][0].w, w4[d][1].w, x4[d][h].z, x4[d][h].w);
        }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int c = 0; c < 4; ++c) sums[warp][g + c / 2 * 8][8 * h + 2 * q + c % 2] = acc[h][c];
    __syncthreads();
    const int i = tid % FEW_RANKS, m = tid / FEW_RANKS;
    if (m < 16 && m0 + m < n && i0 + i < per) {
      float sum = 0.f;
#pragma unroll
      for (int s = 0; s < WARPS; ++s) sum += sums[s][i][m];
      const int part = (i0 + i) / bank.rank, j = (i0 + i) % bank.rank;
      bf16* at = to + (size_t)list[m0 + m] * width + part * bank.wide + j;
      *at = __float2bfloat16_rn(j < bank.ranks[a * bank.parts + part] ? sum * bank.scale[a * bank.parts + part] : 0.f);
      if (j + 8 >= bank.rank && bank.wide > bank.rank) at[8] = __float2bfloat16_rn(0.f);  // the product takes whole steps of sixteen
    }
    __syncthreads();
  }
  if constexpr (!COMPACT)
    for (int o = tid; o < 2 * rows; o += 32 * WARPS) {
      const int i = i0 + o % 2 * 8, r = o / 2;
      if (i >= per || tiles.row_adapter[r] == a) continue;
      bf16* at = to + (size_t)r * width + i / bank.rank * bank.wide + i % bank.rank;
      *reinterpret_cast<uint4*>(at) = zero;
      if (i % bank.rank + 8 == bank.rank && bank.wide > bank.rank) *reinterpret_cast<uint4*>(at + 8) = zero;
    }
}

template <bool COMPACT, int WARPS>
int launch_few(bf16* t, int* done, int n_done, const bf16* x, long long ldx, int K, const AdapterBank& bank, const AdapterTiles& tiles, cudaStream_t stream) {
  const dim3 grid((bank.parts * bank.rank + FEW_RANKS - 1) / FEW_RANKS, min(tiles.n_slots, bank.capacity));
  return (int)launch_pdl(first_factor_few_kernel<COMPACT, WARPS>, grid, dim3(32 * WARPS), 0, stream, t, done, n_done, x, ldx, K, bank, tiles);
}

// rows and ranks of a copy of the first factor's: as many as there are (64 of the ranks where the rows are many: the sums of both have their place in shared memory)
int first_rows(const AdapterTiles& tiles) { return min(128, (min(tiles.rows, tiles.tile_rows) + 7) / 8 * 8); }
int first_ranks(const AdapterBank& bank, const AdapterTiles& tiles) { return min(first_rows(tiles) > 64 ? 64 : FIRST_RANKS, (bank.parts * bank.rank + 15) / 16 * 16); }

int launch_first(bf16* t, int* done, int n_done, const CUtensorMap& map_x, const CUtensorMap& map_a, int K, const AdapterBank& bank, const AdapterTiles& tiles, int* error,
                 cudaStream_t stream) {
  auto kern = first_factor_tiles_kernel;
  // an SM gives its memory to L1 or to blocks anew only when it is empty: split as the product's blocks need it, they come in beside these
  static unsigned long long told = 0, allowed = 0;
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e == cudaSuccess && !(__atomic_load_n(&told, __ATOMIC_RELAXED) >> (device & 63) & 1)) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    if (e == cudaSuccess) __atomic_fetch_or(&told, 1ull << (device & 63), __ATOMIC_RELAXED);
  }
  if (e == cudaSuccess) e = allow_shared(kern, FIRST_DEEP_BYTES, &allowed);
  if (e != cudaSuccess) return (int)e;
  const int row_tiles = (tiles.rows + tiles.tile_rows - 1) / tiles.tile_rows, ranks = bank.parts * bank.rank;
  const int box_rows = first_rows(tiles), box_ranks = first_ranks(bank, tiles);
  const int parts = (min(tiles.tile_rows, tiles.rows) + 127) / 128, chunks = (ranks + box_ranks - 1) / box_ranks;
  // Blocks that share k: of a single tile, whose adapters are in the first slots, as the SMs take one of; of many tiles, of whose slots some third
  // is not used, six at most (clusters of eight leave an eighth of the SMs without one).
  // (By the bank's room: 64 rows of one adapter, 9,728 x 2,560, 28.7 us in a bank of one, 30.8 of 24 and 41 of 64.)
  const int slots = row_tiles == 1 ? min(tiles.n_slots, bank.capacity) : tiles.n_slots;
  const long long blocks = (long long)slots * parts * chunks;
  const int most = row_tiles == 1 ? 8 : 6;
  int ways = (int)max(1ll, min((long long)most, (row_tiles == 1 ? 148 : 180) / blocks));
  ways = max(1, min(ways, K / 128));
  // Beside the product's blocks where these take tiles of few rows and wait for W's bytes; before them, on all of an SM's memory, where they would be slowed
  // down. Products read 128 rows, so that the last stage has them behind it.
  const int stage = (box_rows + box_ranks) * 128, behind = max(0, 128 - box_rows - box_ranks) * 128;
  const int sums = ways * ((box_rows + ways - 1) / ways) * (box_ranks + 4) * 4, inbox = ways > 1 ? sums : 0;
  const int room = (tiles.tile_rows > 128 ? FIRST_DEEP_BYTES : FIRST_BYTES) - 1024 - inbox;
  const int stages = max(1, min(FIRST_STAGES, (room - behind) / stage)), ring = (max(stages * stage + behind, sums - inbox) + 1023) / 1024 * 1024;
  const int bytes = 1024 + ring + inbox;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(slots * ways, parts, chunks);
  cfg.blockDim = dim3(FIRST_THREADS);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ways;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  static const bool plain = getenv("KRK_NO_PDL") != nullptr;
  cfg.attrs = attr;
  cfg.numAttrs = plain ? 1 : 2;
  return (int)cudaLaunchKernelEx(&cfg, kern, t, done, n_done, map_x, map_a, K, bank, tiles, ways, stages, ring, box_rows, box_ranks, error);
}

}  // namespace

int krk_first_factor(void* t, bool compact, int* done, int n_done, const void* x, long long ldx, int K, const AdapterBank& bank, const AdapterTiles& tiles, int* error,
                     cudaStream_t stream) {
  const long long rows = (long long)bank.capacity * bank.parts * bank.rank;
  if (rows > 0x7fffffffLL || (long long)tiles.n_slots * 8 > 0x7fffffffLL) return -3;
  if (compact) return launch_few<true, 16>((bf16*)t, done, n_done, (const bf16*)x, ldx, K, bank, tiles, stream);
  // A tile of more than 128 rows with many slots, which blocks of the other kernel would take all of an SM's memory for, the product's blocks behind them: 256 rows of
  // 9,728 x 2,560 with 120 adapters of rank 16 105 us cold, 61 here; 32 adapters 57 and 55, of 2,560 x 6,144 45 and 37; 160 rows with 64 of rank 64 70 and
  // 53, of 4,096 x 2,560 55 and 64; with eight adapters, of 9,728 x 2,560, 49 and 59. These banks held what the step used. The rule goes by the bank's room, since which
  // adapters a step has is known on the device alone, and loses where few of them have many rows each: 200 rows of one adapter of 9,728 x 2,560 43 in a bank of one, 45 of
  // 23, and 172 of 24 or more; of eight adapters 51 and 59.
  if (tiles.rows <= tiles.tile_rows && tiles.tile_rows > 128 && min(tiles.n_slots, bank.capacity) >= 24)
    return launch_few<false, 8>((bf16*)t, done, n_done, (const bf16*)x, ldx, K, bank, tiles, stream);
  CUtensorMap map_x, map_a;
  int rc = make_map_bf16(&map_x, x, tiles.rows, K, ldx, first_rows(tiles));
  if (!rc) rc = make_map_bf16(&map_a, bank.a, rows, K, K, first_ranks(bank, tiles));
  if (rc) return rc;
  return launch_first((bf16*)t, done, n_done, map_x, map_a, K, bank, tiles, error, stream);
}
