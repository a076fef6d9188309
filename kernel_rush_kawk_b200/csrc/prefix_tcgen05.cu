// The prefix parts of groups of many rows on the 5th-generation tensor cores (partial_attention.cuh says what the parts are): every
// row of a group, of any of its sequences, against every key of the prefix that they share.
//
// Here the rows of a decode step that share a prefix are what a prompt's tokens are: one product. 64 sequences of four heads a kv head are
// 256 rows, which meet each key once: 1,024 D operations for the 4 D bytes of a key and its value, the machine's own balance.
//
// A block owns two tiles of 128 (token, head) rows of one kv head and a share of the prefix's pages; S = Q K^T, P and O live in tensor
// memory, K and V come by TMA, 128 keys (two pages) a step, two stages each:
//   tensor memory (512 columns): S0 | S1 | O0 | O1. P_t, rounded to bfloat16, overwrites the first 64 columns of S_t (two keys per 32-bit
//   column) and is the A operand of O_t += P_t V.
// Warps 0..3 run the softmax of tile 0 and warps 4..7 that of tile 1 (thread = row = tensor-memory lane, all 128 keys of a step); warp 8 issues the
// MMAs, lane 0 of warp 9 the TMA loads. While one tile's rows are in the softmax the tensor core works for the other.
//
// What bounds it: for one pair of tiles what comes before its few steps (tables, first pages, first softmax) and behind them, else the chain of a tile's step, as in the kernel for prompts. The MMAs are
// issued by a whole warp that elects a lane for each: their descriptors then stay in registers that the warp shares. From one
// lane's branch an MMA took 113 clocks to issue, where the tensor core needs 65 to 70, and that was the bound. 64 sequences behind 8,192 positions,
// 32 heads over 8 of 128 (34 MB, 8.6 GFLOP; a pair of tiles a block, three or four steps each): 19.7 us (23.0 from one lane); sixteen questions of up to 90
// tokens behind 4,096 positions (73 GFLOP): 75 us, 977 TFLOP/s (93 from one lane). S of 64 keys in two places a tile, two steps ahead of the softmax, was
// slower: a product of 64 columns takes the tensor core as long as one of 128. Asking for the sequences' own pages ahead into L2 from here gained
// nothing: this kernel slowed down by as much as the next one gained.
//
// A group of no more than one tile (HALVES): both halves of the block have the same rows and take the steps in turn, as parts of their own.
// No row masks a key: only the last step of a share may have a single page, whose missing half takes part in nothing.
//
// The reference maximum m of a row moves only when the row's maximum has grown by more than 2^8 since it was set (its row of O is then
// rescaled in tensor memory); until then p <= 2^8. The part that leaves is (m, sum, O) in float32, with
// whichever m. P in bfloat16 is off by half a step, 2^-8 of a weight.
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
constexpr int ROWS = 128;              // rows per tile
constexpr int KEYS = 128;              // keys per step: two pages
constexpr int DB = D / 64;             // 64-wide blocks of the head dimension
constexpr int THREADS = 384;           // 8 softmax warps, the one that issues the MMAs, the one that loads, two idle
constexpr uint32_t SUB = 128 * 128;    // bytes of a [128 rows x 64 bf16] swizzled sub-tile
constexpr uint32_t TILE_BYTES = DB * SUB;  // a Q, K or V tile
constexpr uint32_t TMEM_COLS = 512;
constexpr uint32_t TMEM_O = 256;       // O_t starts at column 256 + t * D; S_t at t * 128
constexpr float LOG2E = 1.4426950408889634f;
constexpr float RESCALE_STEP = 8.f;    // in log2 units

enum Bar { K_FULL = 0, V_FULL = 2, K_FREE = 4, V_FREE = 6, S_FULL = 8, P_READY = 10, O_LAST = 12, Q_FULL = 14, N_BARS };

__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// byte offset of the 16-byte piece `chunk` (8 elements) of row `r` inside a swizzled [128 x 64] sub-tile
__device__ __forceinline__ uint32_t swz(int r, int chunk) { return (uint32_t)r * 128u + (uint32_t)((chunk ^ (r & 7)) << 4); }

// 32 bytes at once: a whole sector of the row that a thread holds
__device__ __forceinline__ void store_8(float* p, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]),
               "r"(v[6]), "r"(v[7])
               : "memory");
}

__global__ void __launch_bounds__(THREADS, 1)
prefix_tcgen05_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_q,
                      int q_by_tma, int rows, Parts parts, int part0, int n_splits, bool halves, const bf16* __restrict__ q, int q_stride, int HQ, int HKV,
                      Segments seg, float scale_log2, int* __restrict__ error) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* base = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  unsigned char* q_s = base;                        // two tiles
  unsigned char* k_s = q_s + 2 * TILE_BYTES;        // two stages
  unsigned char* v_s = k_s + 2 * TILE_BYTES;        // two stages
  uint64_t* bars = reinterpret_cast<uint64_t*>(v_s + 2 * TILE_BYTES);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + N_BARS);

  // Groups, slots and page tables are written by copies and by kernels that no later one overtakes: read before the wait for the kernel that
  // writes the rows.
  const int kh = blockIdx.x % HKV, split = blockIdx.x / HKV % n_splits, pair = blockIdx.x / HKV / n_splits;
  const int G = HQ / HKV;
  const Unit u = prefix_unit(seg, blockIdx.y);
  const int n_rows = u.n_tok * G, pair_row = pair * 2 * rows;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;  // (a number that the compiler knows to be the warp's)
  int p_lo, p_hi;
  split_pages(0, u.key_hi, split, n_splits, p_lo, p_hi);
  const int n_pages = p_hi - p_lo;
  auto page_row = [&](int p) { return p < n_pages ? (seg.table[(size_t)u.slot * seg.width + p_lo + p] * HKV + kh) * KRK_PAGE : 0; };
  int first_pages[4];
  if (warp == 9)
#pragma unroll
    for (int p = 0; p < 4; ++p) first_pages[p] = page_row(p);
  grid_dependency_wait();
  grid_launch_dependents();  // in this order: the next kernel reads rows and keys before it waits for the parts
  if (pair_row >= n_rows) return;
  const int tiles = halves || pair_row + rows < n_rows ? 2 : 1;
  // tile t's rows start at tile_row(t), its j-th step is block_of(t, j) of the share's n blocks of 128 keys, and it has steps(t) of them
  const int n = (n_pages + 1) / 2;
  const bool odd = n_pages & 1;  // the last block has one page
  auto tile_row = [&](int t) { return pair_row + (halves ? 0 : t * rows); };
  auto block_of = [&](int t, int j) { return halves ? 2 * j + t : j; };
  auto steps = [&](int t) { return t >= tiles ? 0 : halves ? (n + 1 - t) / 2 : n; };
  auto part_of = [&](int t) { return part0 + split + (halves ? t * n_splits : 0); };

  if (n_pages == 0) {  // more splits than pages, or a group that shares nothing
    for (int i = threadIdx.x; i < tiles * rows; i += THREADS) {
      const int t = i / rows, R = tile_row(t) + i % rows;
      if (R < n_rows) parts.ml[parts.at(part_of(t), u.row0 + R / G, kh * G + R % G)] = make_float2(-INFINITY, 0.f);
    }
    return;
  }
  const int q_tiles = halves ? 1 : tiles;

  if (warp == 8) {
    // A block of this step that gave up on a wait (codes from 3 on): the others do no work.
    const int error_now = *reinterpret_cast<volatile int*>(error);
    if (lane == 0) {
      for (int i = 0; i < N_BARS; ++i) mbar_init(bars + i, i == P_READY || i == P_READY + 1 ? ROWS / 32 : 1);
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
      tmem_slot[1] = (uint32_t)(error_now >= 3);
      if (q_by_tma && error_now < 3) {
        // a tile is a box of whole tokens x G heads x 64 dims per 64-wide block of the head: its rows land in (token, head) order
        mbar_expect_tx(bars + Q_FULL, q_tiles * DB * rows * 128);
        for (int t = 0; t < q_tiles; ++t)
#pragma unroll
          for (int h = 0; h < DB; ++h)
            tma_load_3d(q_s + t * TILE_BYTES + h * SUB, &map_q, bars + Q_FULL, h * 64, kh * G, u.row0 + tile_row(t) / G);
      }
    }
  } else if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(TMEM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (!q_by_tma) {
    for (int i = threadIdx.x; i < q_tiles * ROWS * (D / 8); i += THREADS) {
      const int r = i / (D / 8), c = i % (D / 8), R = pair_row + r;  // rows is ROWS here
      uint4 v = make_uint4(0, 0, 0, 0);
      if (R < n_rows) v = *reinterpret_cast<const uint4*>(q + (size_t)(u.row0 + R / G) * q_stride + (size_t)(kh * G + R % G) * D + c * 8);
      *reinterpret_cast<uint4*>(q_s + (r / ROWS) * TILE_BYTES + (c / 8) * SUB + swz(r % ROWS, c % 8)) = v;
    }
    fence_async_smem();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const bool dead = tmem_slot[1] != 0;

  if (dead) {
    // nothing to do
  } else if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == 8) {
      // ---- issuer of the MMAs ----
      // a negative scale: the products leave negated (the descriptor's bit for A), and the softmax takes the scale's size, so that maxima before it
      // are maxima after it
      const uint32_t idesc_s = (scale_log2 < 0.f ? 1u << 13 : 0u) | (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(KEYS >> 3) << 17) | ((uint32_t)(ROWS >> 4) << 24);
      constexpr uint32_t idesc_o = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((uint32_t)(D >> 3) << 17) | ((uint32_t)(ROWS >> 4) << 24);
      // descriptors: what does not change is put together once, and an instruction's own differ from these by their address (in 16 bytes, in
      // the low word, with no carry): the issuing thread's instructions are what a step waits for
      const uint64_t q_desc = umma_desc_sw128(q_s, 16, 1024), k_desc = umma_desc_sw128(k_s, 16, 1024), v_desc = umma_desc_sw128(v_s, SUB, 1024);
      auto moved = [](uint64_t desc, uint32_t by) { return (desc & 0xffffffff00000000ull) | ((uint32_t)desc + by); };
      bool ok = true;
      auto wait = [&](int bar, uint32_t parity, int code) {
        if (ok && !__all_sync(0xffffffffu, mbar_wait(bars + bar, parity))) {
          if (lane == 0) atomicExch(error, code);
          ok = false;
        }
        return ok;
      };
      auto qk = [&](int t, int j) {  // S_t = Q_t K^T of the tile's j-th step
        const int i = block_of(t, j), stage = i & 1;
        if (!wait(K_FULL + stage, (i >> 1) & 1, 10)) return;
        tc_fence_after();
        const uint64_t qd = moved(q_desc, (halves ? 0 : t) * (TILE_BYTES >> 4)), kd = moved(k_desc, stage * (TILE_BYTES >> 4));
#pragma unroll
        for (int h = 0; h < DB; ++h)
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            umma_bf16_warp(tmem + t * 128, moved(qd, h * (SUB >> 4) + kk * 2), moved(kd, h * (SUB >> 4) + kk * 2), idesc_s, (h > 0 || kk > 0) ? 1u : 0u);
        umma_commit_warp(bars + S_FULL + t);
        if (halves || t == tiles - 1) umma_commit_warp(bars + K_FREE + stage);
      };
      auto pv = [&](int t, int j) {  // O_t (+)= P_t V, 16 keys (8 columns of P) per instruction
        const int i = block_of(t, j), stage = i & 1;
        if (!wait(P_READY + t, j & 1, 8) || !wait(V_FULL + stage, (i >> 1) & 1, 9)) return;
        tc_fence_after();
        const uint64_t vd = moved(v_desc, stage * (TILE_BYTES >> 4));
        auto page = [&](int k0) {
#pragma unroll
          for (int kk = k0; kk < k0 + KEYS / 32; ++kk)
            umma_bf16_tmem_a_warp(tmem + TMEM_O + t * D, tmem + t * 128 + kk * 8, moved(vd, kk * (16 * 128 >> 4)), idesc_o, (j == 0 && kk == 0) ? 0u : 1u);
        };
        page(0);
        if (!(odd && i == n - 1)) page(KEYS / 32);  // a page that is not there takes no part: zero times anything
        if (j == steps(t) - 1) umma_commit_warp(bars + O_LAST + t);
        if (halves || t == tiles - 1) umma_commit_warp(bars + V_FREE + stage);
      };
      const int n0 = steps(0), n1 = steps(1);
      if (q_by_tma) wait(Q_FULL, 0, 14);
      if (ok) qk(0, 0);
      if (ok && n1 > 0) qk(1, 0);
#pragma unroll 1
      for (int j = 0; j < n0 && ok; ++j) {
        pv(0, j);
        if (ok && j + 1 < n0) qk(0, j + 1);
        if (ok && j < n1) pv(1, j);
        if (ok && j + 1 < n1) qk(1, j + 1);
      }
    } else if (warp == 9 && lane == 0) {
      // ---- loader ----
      int asked_k = 0, asked_v = 0;
      auto load = [&](unsigned char* dst, const CUtensorMap* map, uint64_t* bar, int row0, int row1, bool half) {
        mbar_expect_tx(bar, half ? TILE_BYTES / 2 : TILE_BYTES);
#pragma unroll
        for (int h = 0; h < DB; ++h) tma_load_2d(dst + h * SUB, map, bar, h * 64, row0);
        if (!half)
#pragma unroll
          for (int h = 0; h < DB; ++h) tma_load_2d(dst + h * SUB + 64 * 128, map, bar, h * 64, row1);
      };
      int r0 = first_pages[0], r1 = first_pages[1], s0 = first_pages[2], s1 = first_pages[3];  // rows of this block's pages and the next one's
      for (int i = 0; i < n; ++i) {
        const int b = i & 1;
        const uint32_t parity = ((i >> 1) - 1) & 1;
        const bool half = odd && i == n - 1;
        const int next0 = page_row(2 * i + 4), next1 = page_row(2 * i + 5);
        if (i >= 2 && !mbar_wait(bars + K_FREE + b, parity)) { atomicExch(error, 11); break; }
        load(k_s + b * TILE_BYTES, &map_k, bars + K_FULL + b, r0, r1, half);
        asked_k = i + 1;
        if (i >= 2 && !mbar_wait(bars + V_FREE + b, parity)) { atomicExch(error, 7); break; }
        load(v_s + b * TILE_BYTES, &map_v, bars + V_FULL + b, r0, r1, half);
        asked_v = i + 1;
        r0 = s0; r1 = s1; s0 = next0; s1 = next1;
      }
      // what was asked for lands before the block ends, whoever gave up
      wait_for_copies(bars + K_FULL, 2, asked_k);
      wait_for_copies(bars + V_FULL, 2, asked_v);
      if (q_by_tma) mbar_wait(bars + Q_FULL, 0);
    }
  } else {
    // a thread keeps its 128 scores in registers: of the 168 that 384 threads start with the softmax warps take 216 each and the others 72
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    // ---- softmax: warps 0..3 have tile 0, warps 4..7 tile 1; thread = row (its tensor-memory lane), whole steps ----
    const int t = warp >> 2, quad = warp & 3, r = quad * 32 + lane;
    const uint32_t lane_addr = (uint32_t)(quad * 32) << 16;
    const uint32_t tmem_o = tmem + TMEM_O + t * D + lane_addr;
    const int R = tile_row(t) + r, my_steps = steps(t);
    const bool valid = r < rows && R < n_rows;  // other threads' scores are anything, decide nothing and go nowhere
    float m = -INFINITY;
    float2 l2 = make_float2(0.f, 0.f);
    const float scale_size = fabsf(scale_log2);
    const float2 scale2 = make_float2(scale_size, scale_size);
    bool ok = true;
    const uint32_t tmem_s = tmem + t * 128 + lane_addr;
    for (int j = 0; j < my_steps; ++j) {
      if (!__all_sync(0xffffffffu, mbar_wait(bars + S_FULL + t, j & 1))) {  // a warp gives up as a whole
        if (lane == 0) atomicExch(error, 12);
        ok = false;
        break;
      }
      tc_fence_after();
      uint32_t s[KEYS];
#pragma unroll
      for (int c = 0; c < KEYS / 32; ++c) tmem_ld_32x32(tmem_s + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(s + 32 * c));
      tmem_wait_ld();
      if (odd && block_of(t, j) == n - 1) {
#pragma unroll
        for (int c = KEYS / 2; c < KEYS; ++c) s[c] = 0xff800000u;  // minus infinity: a key that is not there
      }
      float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int c = 0; c < KEYS; c += 8)
#pragma unroll
        for (int e = 0; e < 4; ++e) mx4[e] = fmaxf(fmaxf(mx4[e], __uint_as_float(s[c + e])), __uint_as_float(s[c + 4 + e]));
      const float m_new = fmaxf(m, fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * scale_size);
      const bool outgrown = valid && m != -INFINITY && m_new - m > RESCALE_STEP;
      if (__any_sync(0xffffffffu, outgrown)) {
        // this step's P V has not been issued and the one before it is complete (this step's S came after it): nothing else touches these rows of O
        const float alpha = m == -INFINITY ? 1.f : fast_exp2(m - m_new);
#pragma unroll 1
        for (int c0 = 0; c0 < D; c0 += 32) {
          uint32_t o[32];
          tmem_ld_32x32(tmem_o + c0, o);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
          tmem_st_32x32(tmem_o + c0, o);
        }
        l2.x *= alpha;
        l2.y *= alpha;
        m = m_new;
      } else if (m == -INFINITY) {
        m = m_new;
      }
      const float m_safe = m == -INFINITY ? 0.f : m;
      const float2 minus_m = make_float2(-m_safe, -m_safe);
      float2 sum = make_float2(0.f, 0.f);  // a step's weights are added up by themselves: one chain over thousands of keys would drift
#pragma unroll
      for (int c0 = 0; c0 < KEYS; c0 += 32) {
        uint32_t pk[16];
#pragma unroll
        for (int c = 0; c < 32; c += 2) {
          const float2 x = __ffma2_rn(make_float2(__uint_as_float(s[c0 + c]), __uint_as_float(s[c0 + c + 1])), scale2, minus_m);
          const float2 p = make_float2(fast_exp2(x.x), fast_exp2(x.y));
          sum = __fadd2_rn(sum, p);
          const __nv_bfloat162 h = __floats2bfloat162_rn(p.x, p.y);
          pk[c / 2] = *reinterpret_cast<const uint32_t*>(&h);
        }
        tmem_st_32x16(tmem_s + c0 / 2, pk);
      }
      l2 = __fadd2_rn(l2, sum);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bars + P_READY + t);
    }
    if (t < tiles && ok) {
      const size_t to = valid ? parts.at(part_of(t), u.row0 + R / G, kh * G + R % G) : 0;
      if (my_steps == 0) {
        if (valid) parts.ml[to] = make_float2(-INFINITY, 0.f);
      } else if (__all_sync(0xffffffffu, mbar_wait(bars + O_LAST + t, 0))) {
        tc_fence_after();
        if (valid) parts.ml[to] = make_float2(m, l2.x + l2.y);
#pragma unroll
        for (int c0 = 0; c0 < D; c0 += 32) {
          uint32_t o[32];
          tmem_ld_32x32(tmem_o + c0, o);
          tmem_wait_ld();
          if (valid)
#pragma unroll
            for (int c = 0; c < 32; c += 8) store_8(parts.o + to * D + c0 + c, o + c);
        }
      } else if (lane == 0) {
        atomicExch(error, 13);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
  }
}

constexpr size_t SMEM_BYTES = 6 * TILE_BYTES + 1024 + N_BARS * 8 + 64;

}  // namespace

// krk_prefix_few_rows for groups of many rows. Rows and pages from 16-byte boundaries on (-2 otherwise); o from 32-byte ones. halves: no group has more
// rows than a tile, and there are twice n_splits parts.
KRK_API int krk_prefix_tcgen05(float* o, float* ml, int rows, int part0, int n_splits, const void* q, int q_stride, int HQ, int HKV, const int* cu_q,
                               const int* seq_slot, const int* seq_start, const int* seq_qlen, const int* group_cu, const int* group_len,
                               const int* seq_group, int n_seqs, int n_groups, const int* table, int width, const void* k_cache, const void* v_cache,
                               int n_pages, int max_rows, int halves, float scale, int* error, cudaStream_t stream) {
  if (rows == 0 || n_groups == 0) return 0;
  if (q_stride % 8 || ((uintptr_t)q & 15) || ((uintptr_t)o & 31)) return -2;
  const int G = HQ / HKV;
  // tiles come by TMA where whole tokens (G rows each) fill most of one; a tile then has that many rows
  const int whole = G <= ROWS ? ROWS / G * G : 0;
  const int q_by_tma = whole >= 112;
  const int tile_rows = q_by_tma ? whole : ROWS;
  if (halves && (long long)max_rows * G > tile_rows) return -2;
  const long long pairs = ((long long)max_rows * G + 2 * tile_rows - 1) / (2 * tile_rows);
  if (pairs * HKV * n_splits > 0x7fffffffLL || n_groups > 65535) return -3;
  CUtensorMap map_k, map_v;
  const long long key_rows = (long long)n_pages * HKV * KRK_PAGE;
  int rc = make_map_bf16(&map_k, k_cache, key_rows, D, D, KRK_PAGE);
  if (rc == 0) rc = make_map_bf16(&map_v, v_cache, key_rows, D, D, KRK_PAGE);
  CUtensorMap map_q = map_k;
  if (rc == 0 && q_by_tma) rc = make_map_bf16_3d(&map_q, q, D, HQ, rows, D, q_stride, G, tile_rows / G);
  if (rc) return rc;
  if (scale == 0.f) scale = 1e-30f;  // a key that is not there has no weight by a score of minus infinity: the scale must not be zero
  static unsigned long long allowed = 0;
  cudaError_t e = allow_shared(prefix_tcgen05_kernel, SMEM_BYTES, &allowed);
  if (e != cudaSuccess) return (int)e;
  const Parts parts = {o, (float2*)ml, rows, HQ};
  const Segments seg = {cu_q, seq_slot, seq_start, seq_qlen, group_cu, group_len, seq_group, n_seqs, n_groups, table, width};
  return (int)launch_pdl(prefix_tcgen05_kernel, dim3((unsigned)(pairs * HKV * n_splits), n_groups), dim3(THREADS), SMEM_BYTES, stream, map_k, map_v, map_q,
                         q_by_tma, tile_rows, parts, part0, n_splits, halves != 0, (const bf16*)q, q_stride, HQ, HKV, seg, scale * LOG2E, error);
}

#endif  // head sizes served by this kernel
