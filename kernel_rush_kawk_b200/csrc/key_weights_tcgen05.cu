// The weight that each key of a sequence receives from a step's queries, on the 5th-generation tensor cores (key_weights_kernel in
// partial_attention.cu has the definition): with the logarithms of the rows' sums known, a key's weight is
//   sum over rows of 2^(k . q scale - lse[row]),
// a sum along the columns of S^T = K Q^T. A block owns 128 keys (two pages) of a kv head, the rows of the accumulator: a thread holds a
// key, reads its scores with 128 rows at a time from tensor memory and adds up, with no exchange between threads, in one order.
//
// The rows that see the keys come by TMA in tiles of whole tokens, two in shared memory; S has two places in tensor memory (256 columns).
// Warps 0..3 take the even tiles and warps 4..7 the odd ones; lane 0 of warp 8 issues the MMAs, lane 0 of warp 9 the loads. Where the blocks
// are few for the device, the tiles of a block's rows are dealt out to a cluster, whose sums meet in the first block, in order; where
// queries are the keys, so that the first keys are seen by every row and the last by few, a block takes a key tile from either end.
//
// What bounds it is the exponentials, one for every (query head, key): 16 a clock and SM, 1,024 clocks a tile; two blocks an SM take 1,010
// to 1,040 a tile between them while both run. (S twice in tensor memory for each half, to read ahead, spilled and was slower; tiles dealt
// to blocks of their own, whose sums a second launch adds, took 9 us more.) Three prompts of up to 1,500 tokens, 12 heads over 4 of 128:
// 29 us, of which 5 a key tile are what comes before its first and behind its last row tile; the last 64 queries of a prompt of 4,001, 32 heads
// over 8: 9.3 us.
//
// Compiled once per head size, for head sizes 64 and 128: -DKRK_HEAD_DIM=<D>.
#include "partial_attention.cuh"
#include "tcgen05.cuh"

#ifndef KRK_HEAD_DIM
#error "compile with -DKRK_HEAD_DIM=<head size>"
#endif

#if KRK_HEAD_DIM == 64 || KRK_HEAD_DIM == 128

namespace {

using namespace tc;

constexpr int D = KRK_HEAD_DIM;
constexpr int ROWS = 128;              // rows (columns of the accumulator) of a tile
constexpr int KEYS = 128;
constexpr int DB = D / 64;
constexpr int THREADS = 320;           // 8 warps that add up, the one that issues, the one that loads
constexpr uint32_t SUB = 128 * 128;    // bytes of a [128 rows x 64 bf16] swizzled sub-tile
constexpr uint32_t TILE_BYTES = DB * SUB;
constexpr uint32_t TMEM_COLS = 256;
constexpr int MAX_SHARE = 8;           // blocks of a cluster
constexpr float LOG2E = 1.4426950408889634f;

enum Bar { K_FULL = 0, Q_FULL = 1, Q_FREE = 3, S_FULL = 5, S_FREE = 7, N_BARS = 9 };

__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__global__ void __launch_bounds__(THREADS, 2)
key_weights_tcgen05_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_q, int rows, const float* sums, float* sums_out,
                           int* __restrict__ positions, const int* __restrict__ seq_shift, int capacity, const float* __restrict__ lse, int observe, int HQ,
                           int HKV, Segments seg, float scale_log2, int share, bool paired, int* __restrict__ error) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* base = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  unsigned char* k_s = base;
  unsigned char* q_s = k_s + TILE_BYTES;  // two stages
  uint64_t* bars = reinterpret_cast<uint64_t*>(q_s + 2 * TILE_BYTES);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + N_BARS + 1);
  float* minus_lse = reinterpret_cast<float*>(tmem_slot + 4);  // [2][ROWS]
  float* other = minus_lse + 2 * ROWS;                         // [KEYS] the odd tiles' sums
  float* inbox = other + KEYS;                                 // [share][KEYS] in the cluster's first block

  if (share > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // "I have started"
  grid_dependency_wait();
  grid_launch_dependents();
  const int rank = blockIdx.x % share, block = blockIdx.x / share;
  const int kh = block % HKV, seq = blockIdx.y, G = HQ / HKV;
  const Unit u = own_unit(seg, seq);
  // key tile a and, of a pair, b: the first with the last, the second with the last but one
  const int key_tiles = (u.key_hi + KEYS - 1) / KEYS, tile_a = block / HKV, tile_b = paired ? key_tiles - 1 - tile_a : tile_a;
  if (tile_a >= key_tiles || tile_a > tile_b) {  // a cluster as a whole
    if (share > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    return;
  }
  const int seen = observe > 0 ? min(observe, u.n_tok) : u.n_tok, tok0 = u.n_tok - seen;
  const int start = u.start + tok0, row0 = u.row0 + tok0, n_rows = seen * G;  // of the rows that count
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (warp == 8) {
    const int error_now = *reinterpret_cast<volatile int*>(error);
    if (lane == 0) {
      for (int i = 0; i < N_BARS; ++i) mbar_init(bars + i, i >= S_FREE ? 4 : 1);
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
      tmem_slot[2] = 0;
      tmem_slot[1] = (uint32_t)(error_now >= 3);  // a kernel of this step gave up on a wait
    }
  } else if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(TMEM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (rows < ROWS) {  // the places behind a tile's rows: zero, so that their scores are numbers
    const int piece = (ROWS - rows) * 8;  // 16-byte pieces of a sub-tile
    for (int i = threadIdx.x; i < 2 * DB * piece; i += THREADS)
      *reinterpret_cast<uint4*>(q_s + (i / piece) * SUB + (size_t)rows * 128 + (i % piece) * 16) = make_uint4(0, 0, 0, 0);
    fence_async_smem();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  if (share > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // every block of the cluster has started

  int done = 0, k_loads = 0;  // row tiles and key tiles of this block so far: the barriers' phases go on
  for (int part = 0; part < (tile_b > tile_a ? 2 : 1); ++part) {
    const int key0 = (part ? tile_b : tile_a) * KEYS;
    const int first = max(0, (key0 - start) * G) / rows + rank;  // of the tiles with a row that sees a key, this block's first
    const int n = max(0, ((n_rows + rows - 1) / rows - first + share - 1) / share);
    const bool half = key0 + KRK_PAGE >= u.key_hi;  // one page only
    const bool dead = tmem_slot[1] != 0 || n == 0;
    auto give_up = [&](int code) {  // the other key tile is not begun
      atomicExch(error, code);
      *reinterpret_cast<volatile uint32_t*>(tmem_slot + 2) = 1;
    };

    float total = 0.f;
    if (dead) {
      // no row sees the keys, or nothing is to be done
    } else if (warp == 8) {
      if (lane == 0) {
        constexpr uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(ROWS >> 3) << 17) | ((uint32_t)(KEYS >> 4) << 24);
        bool ok = mbar_wait(bars + K_FULL, k_loads & 1);
        if (!ok) give_up(6);
        for (int i = done; i < done + n && ok; ++i) {
          const int b = i & 1;
          if (!mbar_wait(bars + Q_FULL + b, (i >> 1) & 1)) { give_up(14); break; }
          if (i >= 2 && !mbar_wait(bars + S_FREE + b, ((i >> 1) - 1) & 1)) { give_up(8); break; }
          tc_fence_after();
          const unsigned char* q = q_s + b * TILE_BYTES;
#pragma unroll
          for (int h = 0; h < DB; ++h)
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              umma_bf16(tmem + b * ROWS, umma_desc_sw128(k_s + h * SUB + kk * 32, 16, 1024), umma_desc_sw128(q + h * SUB + kk * 32, 16, 1024), idesc,
                        (h > 0 || kk > 0) ? 1u : 0u);
          umma_commit(bars + S_FULL + b);
          umma_commit(bars + Q_FREE + b);
        }
      }
    } else if (warp == 9) {
      if (lane == 0) {
        const int* pages = seg.table + (size_t)u.slot * seg.width + key0 / KRK_PAGE;
        mbar_expect_tx(bars + K_FULL, half ? TILE_BYTES / 2 : TILE_BYTES);
        for (int p = 0; p < (half ? 1 : 2); ++p) {
          const int row = (pages[p] * HKV + kh) * KRK_PAGE;
#pragma unroll
          for (int h = 0; h < DB; ++h) tma_load_2d(k_s + h * SUB + p * (64 * 128), &map_k, bars + K_FULL, h * 64, row);
        }
        int asked = done;
        for (int i = done; i < done + n; ++i) {
          const int b = i & 1;
          if (i >= 2 && !mbar_wait(bars + Q_FREE + b, ((i >> 1) - 1) & 1)) { give_up(7); break; }
          mbar_expect_tx(bars + Q_FULL + b, DB * rows * 128);
#pragma unroll
          for (int h = 0; h < DB; ++h)
            tma_load_3d(q_s + b * TILE_BYTES + h * SUB, &map_q, bars + Q_FULL + b, h * 64, kh * G, row0 + (first + (i - done) * share) * rows / G);
          asked = i + 1;
        }
        // what was asked for lands before the block ends, whoever gave up
        mbar_wait(bars + K_FULL, k_loads & 1);
        wait_for_copies(bars + Q_FULL, 2, asked);
      }
    } else {
      const int t = warp >> 2, quad = warp & 3, r = quad * 32 + lane;  // thread = key = tensor-memory lane
      const uint32_t tmem_s = tmem + t * ROWS + ((uint32_t)(quad * 32) << 16);
      const int key = key0 + r;
      const float2 scale2 = make_float2(scale_log2, scale_log2);
      float* mine = minus_lse + t * ROWS;
      bool alive = true;  // false once a wait ran out: the four warps go on to their barriers, the results are void
      // a tile's logarithms are asked for a tile ahead
      auto logarithm = [&](int i) {
        const int R = (first + (i - done) * share) * rows + r;
        return i < done + n && r < rows && R < n_rows ? -lse[(size_t)(row0 + R / G) * HQ + kh * G + R % G] : -INFINITY;
      };
      const int i0 = done + ((t ^ done) & 1);  // even tiles are the first four warps'
      float next = logarithm(i0);
      for (int i = i0; i < done + n; i += 2) {
        const int tile0 = (first + (i - done) * share) * rows;  // the tile's first row, of those that count
        mine[r] = next;
        next = logarithm(i + 2);
        asm volatile("bar.sync %0, 128;" ::"r"(1 + t) : "memory");
        if (alive && !__all_sync(0xffffffffu, mbar_wait(bars + S_FULL + t, (i >> 1) & 1))) {
          if (lane == 0) give_up(12);
          alive = false;
        }
        tc_fence_after();
        // rows from `low` on see the key; rows behind the last are other sequences'
        const int low = (key - start) * G - tile0, high = n_rows - tile0;
        const bool masked = key0 + KEYS - 1 > start + tile0 / G || high < rows;
        float2 acc = make_float2(0.f, 0.f);
#pragma unroll
        for (int c0 = 0; c0 < (alive ? ROWS : 0); c0 += 32) {
          uint32_t s[32];
          tmem_ld_32x32(tmem_s + c0, s);
          tmem_wait_ld();
          if (c0 == ROWS - 32) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bars + S_FREE + t);
          }
          if (masked) {
#pragma unroll
            for (int c = 0; c < 32; ++c)
              if (c0 + c < low || c0 + c >= high) s[c] = 0xff800000u;
#pragma unroll
            for (int c = 0; c < 32; ++c) {
              const float x = __uint_as_float(s[c]) == -INFINITY ? -INFINITY : fmaf(__uint_as_float(s[c]), scale_log2, mine[c0 + c]);
              acc.x += fast_exp2(x);
            }
          } else {
#pragma unroll
            for (int c = 0; c < 32; c += 4) {
              const float4 ml = *reinterpret_cast<const float4*>(mine + c0 + c);
              const float2 x = __ffma2_rn(make_float2(__uint_as_float(s[c]), __uint_as_float(s[c + 1])), scale2, make_float2(ml.x, ml.y));
              const float2 y = __ffma2_rn(make_float2(__uint_as_float(s[c + 2]), __uint_as_float(s[c + 3])), scale2, make_float2(ml.z, ml.w));
              acc = __fadd2_rn(acc, make_float2(fast_exp2(x.x), fast_exp2(x.y)));
              acc = __fadd2_rn(acc, make_float2(fast_exp2(y.x), fast_exp2(y.y)));
            }
          }
        }
        total += acc.x + acc.y;
        asm volatile("bar.sync %0, 128;" ::"r"(1 + t) : "memory");  // the tile's logarithms have been read
      }
      if (t == 1) other[r] = total;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (!dead) {
      done += n;
      ++k_loads;
    }
    const int key = key0 + threadIdx.x;
    if (!dead && threadIdx.x < KEYS) total += other[threadIdx.x];
    if (share > 1) {
      if (threadIdx.x < KEYS)
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(cluster_address(inbox + rank * KEYS + threadIdx.x, 0)), "f"(total) : "memory");
      cluster_sync();
      if (rank == 0 && threadIdx.x < KEYS) {
        total = 0.f;
        for (int c = 0; c < share; ++c) total += inbox[c * KEYS + threadIdx.x];
      }
    }
    if (rank == 0 && threadIdx.x < KEYS && key < u.key_hi) {
      const size_t place = ((size_t)u.slot * HKV + kh) * capacity + key;
      sums_out[place] = key < u.start ? sums[place] + total : total;
      if (positions && key >= u.start) positions[place] = key + (seq_shift ? seq_shift[seq] : 0);
    }
    if (part == 0 && tile_b > tile_a) {
      if (threadIdx.x == 0 && tmem_slot[2]) tmem_slot[1] = 1;
      __syncthreads();  // the odd tiles' sums have been read
      if (share > 1) cluster_sync();  // and what the cluster sent
    }
  }
  if (warp == 9) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
}

constexpr size_t SMEM_BYTES = 3 * TILE_BYTES + 1024 + (N_BARS + 1) * 8 + 16 + (2 * ROWS + (1 + MAX_SHARE) * KEYS) * sizeof(float);

}  // namespace

// krk_key_weights on the tensor cores. max_seen: the most queries of a sequence that count; max_kv_len: the most rows that one holds after the step. -2: rows off 16-byte boundaries, or heads of
// which whole tokens do not fill half a tile.
KRK_API int krk_key_weights_tcgen05(const float* sums, float* sums_out, int* positions, const int* seq_shift, int capacity, const float* lse, int observe,
                                    const void* q, int q_stride, int HQ, int HKV, const int* cu_q, const int* seq_slot, const int* seq_start,
                                    const int* seq_qlen, const int* group_cu, const int* group_len, const int* seq_group, int n_seqs, int n_groups,
                                    const int* table, int width, const void* k_cache, int n_pages, int rows, int max_seen, int max_kv_len, float scale,
                                    int* error, cudaStream_t stream) {
  if (n_seqs == 0 || rows == 0) return 0;
  const int G = HQ / HKV, tile_rows = G <= ROWS ? ROWS / G * G : 0;
  if (q_stride % 8 || ((uintptr_t)q & 15) || tile_rows < ROWS / 2) return -2;
  // Where a sequence's queries are its keys, the first keys are seen by every row and the last by few: key tiles go in pairs of equal work, where they are
  // enough (with the attention, us, one by one and in pairs: a prompt of 4,001 tokens, 32 heads over 8 of 128: 287 and 257; 2,000 beside 1,000: 143
  // and 117; eight of 500: 83.5 and 79; 2,000: 91 and 89; three of up to 1,500, 12 heads over 4: 63.7 and 62.3; but 700, 12 heads over 4: 31.5 and 37.4, 1,000 behind
  // 900: 72 and 76: a second key tile costs its latencies again).
  const long long key_tiles = ((long long)max_kv_len + KEYS - 1) / KEYS, row_tiles = ((long long)max_seen * G + tile_rows - 1) / tile_rows;
  const bool paired = row_tiles >= 8 && 4LL * max_seen >= 3LL * max_kv_len && key_tiles * HKV * n_seqs >= 80;
  const long long blocks = (paired ? (key_tiles + 1) / 2 : key_tiles) * HKV;
  if (blocks * MAX_SHARE > 0x7fffffffLL || n_seqs > 65535) return -3;
  // shares of four tiles or more, no more blocks than run at once (three prompts of up to 1,500 tokens, 12 heads: 44.6 us alone, 31.0 in
  // pairs, 31.6 in fours, 40.3 in eights)
  int share = 1;
  while (share < MAX_SHARE && blocks * n_seqs * 2 * share <= 2 * 148 && row_tiles >= 8 * share) share *= 2;
  CUtensorMap map_k, map_q;
  int rc = make_map_bf16(&map_k, k_cache, (long long)n_pages * HKV * KRK_PAGE, D, D, KRK_PAGE);
  if (rc == 0) rc = make_map_bf16_3d(&map_q, q, D, HQ, rows, D, q_stride, G, tile_rows / G);
  if (rc) return rc;
  static unsigned long long allowed = 0;
  cudaError_t e = allow_shared(key_weights_tcgen05_kernel, SMEM_BYTES, &allowed);
  if (e != cudaSuccess) return (int)e;
  const Segments seg = {cu_q, seq_slot, seq_start, seq_qlen, group_cu, group_len, seq_group, n_seqs, n_groups, table, width};
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(blocks * share), n_seqs);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = SMEM_BYTES;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = share;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return (int)cudaLaunchKernelEx(&cfg, key_weights_tcgen05_kernel, map_k, map_q, tile_rows, sums, sums_out, positions, seq_shift, capacity, lse, observe, HQ,
                                 HKV, seg, scale * LOG2E, share, paired, error);
}

#endif  // head sizes served by this kernel
