#include <cooperative_groups.h>

#include "adapters.cuh"
#include "mma.cuh"
#include "warp_copies.cuh"

namespace {

using namespace tc;

// The first factor of many requests' adapters, t = scale (x A^T), sums in 32 bits on the tensor cores. rounded to bfloat16. Two forms of t: of every slot,
// [slot][tile_rows][parts * wide], zeros where a row has another adapter than the slot's (COMPACT false); of every row, [rows][parts * wide], where it has an adapter. A cluster has 128 rows of a slot's tile (y), 128 of the
// adapter's ranks, all parts' side by side (z), and its `ways` blocks share k. A block multiplies its part of k on the tensor cores (128 rows by 128
// ranks, fed by TMA in blocks of 64 k); the blocks' sums meet in 32 bits through distributed shared memory, each block adding and writing its share of
// the rows, in the blocks' order.
//
// The product's blocks come in while these run, once what came before is over, and wait for t where they need it; so a ring of few blocks of k is no
// larger than fits beside theirs.
constexpr int FIRST_RANKS = 128, FIRST_STAGES = 8, FIRST_THREADS = 192, FIRST_PITCH = FIRST_RANKS + 4;
constexpr int FIRST_BYTES = 72 * 1024;  // of the ring, beside the product's
constexpr int FIRST_BLOCKS = 148;  // as many as are worth sharing k among
static_assert(128 * FIRST_PITCH * 4 <= FIRST_BYTES, "the sums take the ring's place");

template <bool COMPACT>
__global__ void __launch_bounds__(FIRST_THREADS, 5)  // (of three that an SM's memory takes: in 64 registers they fit beside the product's)
first_factor_tiles_kernel(bf16* __restrict__ t, int* __restrict__ done, int n_done, const __grid_constant__ CUtensorMap map_x,
                                                                           const __grid_constant__ CUtensorMap map_a, int K,
                                                                           const __grid_constant__ AdapterBank bank, const __grid_constant__ AdapterTiles tiles,
                                                                           int ways, int stages, int box_rows, int box_ranks, int* __restrict__ error) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* ring = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  float* sums = reinterpret_cast<float*>(ring);  // [128][FIRST_PITCH], when the ring has done its work
  __shared__ uint64_t full_bar[FIRST_STAGES], empty_bar[FIRST_STAGES], acc_bar;
  __shared__ uint32_t tmem_slot;
  __shared__ int asked_for;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, way = blockIdx.x % ways, slot = blockIdx.x / ways;
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
  auto leave = [&] {
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(acc), "r"(FIRST_RANKS) : "memory");
  };
  if (blockIdx.x + blockIdx.y + blockIdx.z == 0)
    for (int i = threadIdx.x; i < n_done; i += FIRST_THREADS) done[i] = 0;  // the product's counts of shares
  const int2 is = *reinterpret_cast<const int2*>(tiles.slots + 2 * slot);
  const int a = is.x, r0 = is.y * tiles.tile_rows + blockIdx.y * 128;
  if (a < 0 || a >= bank.capacity) return leave();  // the whole cluster (the product says so)
  const int here = min(128, min(tiles.tile_rows - (int)blockIdx.y * 128, tiles.rows - r0));  // rows
  if (here <= 0) return leave();
  bool has = false;
  for (int r = threadIdx.x; r < here; r += FIRST_THREADS) has |= tiles.row_adapter[r0 + r] == a;
  const int k_blocks = (K + 63) / 64, each = (k_blocks + ways - 1) / ways, b0 = min(way * each, k_blocks), b1 = min(b0 + each, k_blocks);
  const int n0 = blockIdx.z * FIRST_RANKS, per_adapter = bank.parts * bank.rank;
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
      for (int b = b0; b < b1; ++b) {
        const int i = b - b0, s = i % stages;
        if (i >= stages && !__all_sync(0xffffffffu, mbar_wait(empty_bar + s, (i / stages - 1) & 1))) {
          if (lane == 0) {
            atomicExch(error, 3);
            asked_for = i;
          }
          break;
        }
        const uint32_t stage = smem_u32(ring) + s * bytes, bar = smem_u32(full_bar + s);
        mbar_expect_tx_warp(bar, bytes);
        tma_load_2d_warp(stage, &map_x, bar, b * 64, r0);
        tma_load_2d_warp(stage + box_rows * 128, &map_a, bar, b * 64, a * per_adapter + n0);
      }
    } else if (warp == 1) {
      const uint32_t idesc = umma_idesc(128, box_ranks);  // (rows beyond the copies' give rows that nobody reads)
      for (int b = b0; b < b1; ++b) {
        const int i = b - b0, s = i % stages;
        if (!__all_sync(0xffffffffu, mbar_wait(full_bar + s, (i / stages) & 1))) {
          if (lane == 0) atomicExch(error, 4);
          break;
        }
        tc_fence_after();
        const uint64_t x_desc = umma_desc(ring + s * bytes), a_desc = umma_desc(ring + s * bytes + box_rows * 128);
#pragma unroll
        for (int k = 0; k < 4; ++k) umma_bf16_warp(acc, x_desc + k * 2, a_desc + k * 2, idesc, (b > b0 || k > 0) ? 1u : 0u);
        umma_commit_warp(empty_bar + s);
      }
      umma_commit_warp(&acc_bar);  // arrives even after a failed wait, so that all move on
    }
    if (!__all_sync(0xffffffffu, mbar_wait(&acc_bar, 0)) && lane == 0) atomicExch(error, 5);
    __syncthreads();  // the ring has been read by the products that the barrier stands for
    if (threadIdx.x == 0 && asked_for >= 0)  // copies on their way end before the ring is written
      for (int i = max(0, asked_for - stages); i < asked_for; ++i) mbar_wait(full_bar + i % stages, (uint32_t)(i / stages) & 1u, WAIT_LIMIT_NS / 20);
    __syncthreads();
    if (warp >= 2 && (warp & 3) * 32 < here) {
      const int row = (warp & 3) * 32 + lane;
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < FIRST_RANKS; c += 32) {
        if (c >= box_ranks) break;
        uint32_t v[32];
        tmem_ld_32x32(acc + ((uint32_t)((warp & 3) * 32) << 16) + c, v);
        tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < 32; j += 4)
          *reinterpret_cast<float4*>(sums + row * FIRST_PITCH + c + j) =
              b1 > b0 ? make_float4(__uint_as_float(v[j]), __uint_as_float(v[j + 1]), __uint_as_float(v[j + 2]), __uint_as_float(v[j + 3])) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
      tc_fence_before();
    }
    __syncthreads();
    tc_fence_after();
  }
  leave();  // (nobody who holds tensor memory waits for another block)
  if (has && ways > 1) cluster_sync();
  if (COMPACT && !has) return;
  // eight ranks of a row a thread
  namespace cg = cooperative_groups;
  const int share = (here + ways - 1) / ways, first_row = way * share, rows = min(share, here - first_row);
  const int width = bank.parts * bank.wide;
  for (int o = threadIdx.x; o < rows * (FIRST_RANKS / 8); o += FIRST_THREADS) {
    const int row = first_row + o / (FIRST_RANKS / 8), c = o % (FIRST_RANKS / 8) * 8, part = (n0 + c) / bank.rank, j = (n0 + c) % bank.rank;
    if (part >= bank.parts) continue;
    uint4 pack = make_uint4(0, 0, 0, 0);
    if (tiles.row_adapter[r0 + row] == a) {
      const int rank = bank.ranks[a * bank.parts + part];
      const float scale = bank.scale[a * bank.parts + part];
      float v[8] = {};
      for (int w0 = 0; w0 < ways; w0 += 4) {  // four blocks' on their way at once
        float4 lo[4], hi[4];
#pragma unroll
        for (int w = 0; w < 4; ++w)
          if (w0 + w < ways) {
            const float* from = (ways > 1 ? cg::this_cluster().map_shared_rank(sums, w0 + w) : sums) + row * FIRST_PITCH + c;
            lo[w] = *reinterpret_cast<const float4*>(from);
            hi[w] = *reinterpret_cast<const float4*>(from + 4);
          }
#pragma unroll
        for (int w = 0; w < 4; ++w)
          if (w0 + w < ways) {
            v[0] += lo[w].x; v[1] += lo[w].y; v[2] += lo[w].z; v[3] += lo[w].w;
            v[4] += hi[w].x; v[5] += hi[w].y; v[6] += hi[w].z; v[7] += hi[w].w;
          }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = j + i < rank ? v[i] * scale : 0.f;
      pack = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
    }
    else if (COMPACT) continue;
    bf16* to = t + (COMPACT ? (size_t)(r0 + row) : (size_t)slot * tiles.tile_rows + blockIdx.y * 128 + row) * width + part * bank.wide + j;
    *reinterpret_cast<uint4*>(to) = pack;
    if (j + 8 == bank.rank && bank.wide > bank.rank) *reinterpret_cast<uint4*>(to + 8) = make_uint4(0, 0, 0, 0);  // the product takes whole steps of sixteen
  }
  if (has && ways > 1) cluster_sync();  // no block leaves while another reads its sums
}

// rows and ranks of a copy of the first factor's: as many as there are
int first_rows(const AdapterTiles& tiles) { return min(128, (min(tiles.rows, tiles.tile_rows) + 7) / 8 * 8); }
int first_ranks(const AdapterBank& bank) { return min(FIRST_RANKS, (bank.parts * bank.rank + 15) / 16 * 16); }

template <bool COMPACT>
int launch_first(bf16* t, int* done, int n_done, const CUtensorMap& map_x, const CUtensorMap& map_a, int K, const AdapterBank& bank, const AdapterTiles& tiles, int* error,
                 cudaStream_t stream) {
  auto kern = first_factor_tiles_kernel<COMPACT>;
  // an SM gives its memory to L1 or to blocks anew only when it is empty: split as the product's blocks need it, they come in beside these
  static unsigned long long told = 0, allowed = 0;
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e == cudaSuccess && !(__atomic_load_n(&told, __ATOMIC_RELAXED) >> (device & 63) & 1)) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    if (e == cudaSuccess) __atomic_fetch_or(&told, 1ull << (device & 63), __ATOMIC_RELAXED);
  }
  if (e == cudaSuccess) e = allow_shared(kern, 1024 + FIRST_BYTES, &allowed);
  if (e != cudaSuccess) return (int)e;
  const int row_tiles = (tiles.rows + tiles.tile_rows - 1) / tiles.tile_rows, ranks = bank.parts * bank.rank;
  const int parts = (min(tiles.tile_rows, tiles.rows) + 127) / 128, chunks = (ranks + FIRST_RANKS - 1) / FIRST_RANKS;
  // a single tile's adapters are in the first slots
  const int slots = row_tiles == 1 ? min(tiles.n_slots, bank.capacity) : tiles.n_slots;
  const long long blocks = (long long)slots * parts * chunks;
  int ways = 1;
  while (ways < 8 && 2 * ways * blocks <= FIRST_BLOCKS && K >= 64 * 2 * ways) ways *= 2;
  // Products read 128 rows, so that the last stage has them behind it.
  const int stage = (first_rows(tiles) + first_ranks(bank)) * 128, behind = (128 - first_rows(tiles)) * 128;
  const int stages = min(FIRST_STAGES, (FIRST_BYTES - behind) / stage);
  const int bytes = 1024 + max(stages * stage + behind, 128 * FIRST_PITCH * 4);
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
  return (int)cudaLaunchKernelEx(&cfg, kern, t, done, n_done, map_x, map_a, K, bank, tiles, ways, stages, first_rows(tiles), first_ranks(bank), error);
}

}  // namespace

int krk_first_factor(void* t, bool compact, int* done, int n_done, const void* x, long long ldx, int K, const AdapterBank& bank, const AdapterTiles& tiles, int* error,
                     cudaStream_t stream) {
  const long long rows = (long long)bank.capacity * bank.parts * bank.rank;
  if (rows > 0x7fffffffLL || (long long)tiles.n_slots * 8 > 0x7fffffffLL) return -3;
  CUtensorMap map_x, map_a;
  int rc = make_map_bf16(&map_x, x, tiles.rows, K, ldx, first_rows(tiles));
  if (!rc) rc = make_map_bf16(&map_a, bank.a, rows, K, K, first_ranks(bank));
  if (rc) return rc;
  return compact ? launch_first<true>((bf16*)t, done, n_done, map_x, map_a, K, bank, tiles, error, stream)
                 : launch_first<false>((bf16*)t, done, n_done, map_x, map_a, K, bank, tiles, error, stream);
}
