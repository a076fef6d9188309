// Attention in parts for few rows a unit, bfloat16, on the warp-level tensor cores (partial_attention.cuh says what the parts are):
// a sequence's single token over its own keys, joined with the parts of the prefix that it shares and, where asked for, with
// the weight of each key added up in the same launch; and the prefix parts themselves for groups of few rows.
//
// A block takes 16 rows (the heads of a kv head, or those of several sequences of a group) and a share of the unit's pages; its
// four warps take 16 keys of every page each, with running statistics of their own that join in shared memory at the end. What
// bounds it is the bytes in flight: a unit of work reads D * 256 bytes a page and kv head and multiplies little, so pages come by TMA
// (a fifth warp asks for them, one unit a page of keys or of values, into a ring as deep as the shared memory that
// the blocks of an SM have between them), or by cp.async where the head size is no multiple of 64.
//
// Where a unit has at most eight rows (NARROW: the heads of a kv head mostly are), the products are taken the other way round: the page's
// keys are the sixteen rows of an instruction and the queries its eight columns, S^T = K Q^T and O^T = V^T P^T, with P^T turned in
// registers (movmatrix). Sixteen rows of which four are queries cost twice the instructions and registers:
// 64 sequences' own keys (up to 500 each, 8 kv heads of 128, 70 MB) take 17.2 us in columns and 25.0 in rows, with 96 registers a thread instead of 158 to
// 168. 32 sequences of 2,000 to 4,500 keys with their weights, 8 kv heads of 128: 83 us for 434 MB, 5.2 TB/s, beside 1,631 in the kernel for every type; one
// sequence of 1,087 keys: 8.0 us, the latency of two launches' worth of dependent steps (page table, pages, statistics, join, weights).
//
// The splits of a sequence's keys form a cluster: their parts meet in the first block's shared memory, which also reads the prefix
// parts of its rows and writes the output. That is the only place that waits for the kernel before, so a sequence's own
// keys are read while the prefix kernel still runs.
//
// Weights per key: scaled scores (log2 units, float32) go to scratch as they come, four bytes beside the 4 D that a key costs; when the
// row's sum is known every block of the cluster turns its own keys' scores into weights, sums them over the heads in order
// and adds them to the keys' sums. A key belongs to one thread: no atomics, the same bits every time.
//
// P is rounded to bfloat16 before it meets the values, as everywhere on this path (half a step is 2^-8 of a weight, and errors
// of the keys add up like their weights: far below the output's own rounding); scores, statistics and sums are float32.
//
// Compiled once per head size: -DKRK_HEAD_DIM=<D>.
#include <cooperative_groups.h>

#include "mma.cuh"
#include "partial_attention.cuh"
#include "tcgen05.cuh"

#ifndef KRK_HEAD_DIM
#error "compile with -DKRK_HEAD_DIM=<head size>"
#endif

#if KRK_HEAD_DIM % 16 == 0 && KRK_HEAD_DIM <= 256

namespace {

#include "attention_tiles.cuh"

namespace cg = cooperative_groups;

constexpr int UNIT_ELEMS = TMA_PAGES ? KRK_PAGE * D : TILE_ELEMS;  // one page of keys (or of values) of one kv head
constexpr uint32_t UNIT_BYTES = UNIT_ELEMS * 2;
constexpr int RP = D + 2;  // floats of a row's part in shared memory: o, m, l
constexpr size_t RED_BYTES = (size_t)4 * 16 * RP * sizeof(float);
constexpr int CP_STAGES = 2;  // page pairs, where pages come by cp.async

__device__ __forceinline__ void consumer_sync() { asm volatile("bar.sync 2, 128;" ::: "memory"); }

// The 8 x 8 matrix of bfloat16 pairs that a warp holds, turned.
__device__ __forceinline__ uint32_t turned(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// A warp's running softmax over 16 keys of each page, for 16 rows of queries: S in rows, as in the other kernels of this library.
struct Wide {
  static constexpr int TILE = 16;
  uint32_t qf[KSTEPS][4];
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  float o[DTILES][4], s[2][4];
  __device__ __forceinline__ void begin(const bf16* const (&qp)[2], int lane) {
    load_q(qf, qp[0], qp[1], lane);
#pragma unroll
    for (int n = 0; n < DTILES; ++n)
#pragma unroll
      for (int c = 0; c < 4; ++c) o[n][c] = 0.f;
  }
  template <bool TMA> __device__ __forceinline__ void scores(const bf16* ks, int key0, int count, float scale_log2, int lane) {
    qk_tile<2, TMA>(s, qf, ks, key0, lane);
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int c = 0; c < 4; ++c) s[n][c] = key0 + n * 8 + 2 * (lane & 3) + (c & 1) < count ? s[n][c] * scale_log2 : -INFINITY;
  }
  __device__ __forceinline__ void keep_scores(float* raw, size_t capacity, int q_rows, int lane) const {  // raw: of row 0, the warp's first key
    const int g = lane >> 2, t4 = lane & 3;
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (g + 8 * h < q_rows)
#pragma unroll
        for (int n = 0; n < 2; ++n) *reinterpret_cast<float2*>(raw + (g + 8 * h) * capacity + n * 8 + 2 * t4) = make_float2(s[n][2 * h], s[n][2 * h + 1]);
  }
  __device__ __forceinline__ void update(int) { softmax_update<2>(s, m, l, o); }
  template <bool TMA> __device__ __forceinline__ void values(const bf16* vs, int key0, int lane) { pv_tile<2, TMA>(o, s, vs, key0, lane); }
  __device__ __forceinline__ void leave(float* red, int lane) {  // [16 rows][RP]
    const int g = lane >> 2, t4 = lane & 3;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float* dst = red + (g + 8 * h) * RP;
      if (t4 == 0) { dst[D] = m[h]; dst[D + 1] = l[h]; }
#pragma unroll
      for (int n = 0; n < DTILES; ++n) *reinterpret_cast<float2*>(dst + n * 8 + 2 * t4) = make_float2(o[n][2 * h], o[n][2 * h + 1]);
    }
  }
};

// The same for eight rows of queries, as the columns: a thread has keys g and g + 8 with rows 2 t4 and 2 t4 + 1. The reference maximum of
// a row moves only when it has been outgrown by 2^8 (l and o are float32, P's bfloat16 is relative): then p <= 2^8, and most pages need
// one vote of the warp instead of a maximum over its lanes.
struct Narrow {
  static constexpr int TILE = 8;
  uint32_t qb[KSTEPS][2];
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};  // l: this thread's keys alone, until the end
  float o[KSTEPS][4], s[4];
  __device__ __forceinline__ void begin(const bf16* const (&qp)[2], int lane) {
    const int t4 = lane & 3;
#pragma unroll
    for (int kk = 0; kk < KSTEPS; ++kk) {
      qb[kk][0] = qp[0] ? *reinterpret_cast<const uint32_t*>(qp[0] + kk * 16 + 2 * t4) : 0u;
      qb[kk][1] = qp[0] ? *reinterpret_cast<const uint32_t*>(qp[0] + kk * 16 + 2 * t4 + 8) : 0u;
#pragma unroll
      for (int c = 0; c < 4; ++c) o[kk][c] = 0.f;
    }
  }
  template <bool TMA> __device__ __forceinline__ void scores(const bf16* ks, int key0, int count, float scale_log2, int lane) {
    float odd[4] = {0.f, 0.f, 0.f, 0.f};  // even and odd steps apart: two chains of dependent products
#pragma unroll
    for (int c = 0; c < 4; ++c) s[c] = 0.f;
#pragma unroll
    for (int kk = 0; kk < KSTEPS; ++kk) {
      uint32_t a0, a1, a2, a3;
      ldmatrix_x4(a0, a1, a2, a3, ks + page_off<TMA>(key0 + (lane & 15), kk * 2 + (lane >> 4)));
      mma_bf16_16816(kk & 1 ? odd : s, a0, a1, a2, a3, qb[kk][0], qb[kk][1]);
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) s[c] = key0 + (lane >> 2) + 8 * (c >> 1) < count ? (s[c] + odd[c]) * scale_log2 : -INFINITY;
  }
  __device__ __forceinline__ void keep_scores(float* raw, size_t capacity, int q_rows, int lane) const {
    const int g = lane >> 2, t4 = lane & 3;
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (2 * t4 + (c & 1) < q_rows) raw[(2 * t4 + (c & 1)) * capacity + g + 8 * (c >> 1)] = s[c];
  }
  __device__ __forceinline__ void update(int) {
    // (a NaN outgrows nothing and goes through the sums; rows of infinities come out as they do with a running maximum)
    const bool outgrown = s[0] > m[0] + 8.f || s[2] > m[0] + 8.f || s[1] > m[1] + 8.f || s[3] > m[1] + 8.f;
    if (__any_sync(0xffffffffu, outgrown)) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float mx = fmaxf(s[j], s[2 + j]);
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
        const float m_new = fmaxf(m[j], mx), alpha = m[j] == m_new ? 1.f : fast_exp2(m[j] - m_new);
        m[j] = m_new;
        l[j] *= alpha;
#pragma unroll
        for (int kk = 0; kk < KSTEPS; ++kk) { o[kk][j] *= alpha; o[kk][2 + j] *= alpha; }
      }
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const float ref = m[c & 1];
      s[c] = fast_exp2(s[c] - (ref == -INFINITY ? 0.f : ref));
      l[c & 1] += s[c];
    }
  }
  template <bool TMA> __device__ __forceinline__ void values(const bf16* vs, int key0, int lane) {
    const uint32_t b0 = turned(pack_bf16x2(s[0], s[1])), b1 = turned(pack_bf16x2(s[2], s[3]));
#pragma unroll
    for (int kk = 0; kk < KSTEPS; ++kk) {
      uint32_t a0, a1, a2, a3;
      ldmatrix_x4_trans(a0, a1, a2, a3, vs + page_off<TMA>(key0 + (lane & 7) + ((lane >> 4) << 3), kk * 2 + ((lane >> 3) & 1)));
      mma_bf16_16816(o[kk], a0, a1, a2, a3, b0, b1);
    }
  }
  __device__ __forceinline__ void leave(float* red, int lane) {
    const int g = lane >> 2, t4 = lane & 3;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) l[j] += __shfl_xor_sync(0xffffffffu, l[j], x);
      float* dst = red + (2 * t4 + j) * RP;
      if (g == 0) { dst[D] = m[j]; dst[D + 1] = l[j]; }
#pragma unroll
      for (int kk = 0; kk < KSTEPS; ++kk) {
        dst[kk * 16 + g] = o[kk][j];
        dst[kk * 16 + g + 8] = o[kk][2 + j];
      }
    }
  }
};

struct KeySums {  // weights per key; see krk_scored_single
  float* raw;     // [n_seqs][HQ][capacity]
  const float* sums;
  float* sums_out;
  int* positions;
  const int* seq_shift;
  int capacity;
};

struct Layout {  // of the dynamic shared memory, from a 1024-byte boundary on
  size_t ring, inbox, bars, total;
  __host__ __device__ Layout(int units, int splits, int inbox_rows) {
    ring = 0;
    const size_t r = (size_t)units * UNIT_BYTES;
    inbox = r > RED_BYTES ? r : RED_BYTES;
    inbox = (inbox + 15) & ~(size_t)15;
    bars = inbox + (size_t)(splits > 1 ? splits : 0) * inbox_rows * RP * sizeof(float);
    bars = (bars + 15) & ~(size_t)15;
    total = bars + (size_t)units * 16 + 16 * sizeof(float);
  }
};

// PREFIX: unit = group, parts go to `parts` from part0 on. Otherwise: unit = sequence, one token; the parts 0 .. n_join - 1 of its row join.
template <bool TMA, bool PREFIX, bool SUMS, typename Rows>
__global__ void __launch_bounds__(TMA ? 160 : 128)
few_rows_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, bf16* __restrict__ out, Parts parts, int part0,
                int n_join, const bf16* __restrict__ q, int q_stride, int HQ, int HKV, Segments seg, const bf16* __restrict__ k_cache,
                const bf16* __restrict__ v_cache, float scale_log2, int row_tiles, int units_in_ring, bool wait_first, KeySums ks, int* __restrict__ error) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* base = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  cg::cluster_group cluster = cg::this_cluster();
  const int n_splits = gridDim.x, split = blockIdx.x;
  const bool clustered = !PREFIX && n_splits > 1;
  constexpr int TILE = Rows::TILE;
  const int G = HQ / HKV, inbox_rows = min(TILE, G);
  const Layout at(units_in_ring, clustered ? n_splits : 1, inbox_rows);
  bf16* ring_s = reinterpret_cast<bf16*>(base);
  float* red = reinterpret_cast<float*>(base);            // [4 warps][16 rows][RP], when the ring is done with
  float* inbox = reinterpret_cast<float*>(base + at.inbox);  // [splits][inbox_rows][RP] in the first block
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(base + at.bars);
  uint64_t* empty_bar = full_bar + units_in_ring;
  float* lse_s = reinterpret_cast<float*>(empty_bar + units_in_ring);  // [16]

  if (clustered) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // "I have started"
  if (wait_first) grid_dependency_wait();
  grid_launch_dependents();
  const int kh = blockIdx.y / row_tiles, rt = blockIdx.y % row_tiles;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2;
  const Unit u = PREFIX ? prefix_unit(seg, blockIdx.z) : own_unit(seg, blockIdx.z);
  const int n_rows = u.n_tok * G;
  const int q_rows = min(TILE, n_rows - rt * TILE);
  if (PREFIX && q_rows <= 0) return;  // a whole block, which has asked for nothing
  int j_lo, j_hi;
  split_pages(u.key_lo, u.key_hi, split, n_splits, j_lo, j_hi);
  const int n_pages = j_hi - j_lo;

  if (TMA) {
    if (threadIdx.x == 0) {
      for (int r = 0; r < units_in_ring; ++r) {
        tc::mbar_init(full_bar + r, 1);
        tc::mbar_init(empty_bar + r, 4);
      }
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    if (warp == 4) {
      // ---- the warp that asks for pages: keys and values of a page in turn ----
      int page_here = 0;
      int asked = 0;
      bool ok = true;
      for (int i = 0; i < n_pages && ok; ++i) {
        if (i % 32 == 0) page_here = i + lane < n_pages ? seg.table[(size_t)u.slot * seg.width + j_lo + i + lane] : 0;
        const int page = __shfl_sync(0xffffffffu, page_here, i % 32);
        if (lane == 0) {
          const int row = (page * HKV + kh) * KRK_PAGE;
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int n = 2 * i + half, r = n % units_in_ring;
            if (ok && n >= units_in_ring && !tc::mbar_wait(empty_bar + r, (uint32_t)((n / units_in_ring) - 1) & 1)) {
              atomicExch(error, 25);
              ok = false;
            }
            if (!ok) break;
            tc::mbar_expect_tx(full_bar + r, UNIT_BYTES);
            bf16* dst = ring_s + (size_t)r * UNIT_ELEMS;
#pragma unroll
            for (int h = 0; h < D / 64; ++h) tc::tma_load_2d(dst + h * SUB_ELEMS, half ? &map_v : &map_k, full_bar + r, h * 64, row);
            asked = n + 1;
          }
        }
        ok = __shfl_sync(0xffffffffu, ok, 0);
      }
      if (lane == 0 && !ok) tc::wait_for_copies(full_bar, units_in_ring, asked);  // what was asked for lands before the block ends
      __syncwarp();
      if (clustered) {  // the cluster's barriers count every thread
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        cluster.sync();
        if (SUMS) cluster.sync();
      }
      return;
    }
  }

  // ---- warps 0..3 ----
  const bf16* qp[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int R = rt * TILE + g + 8 * h;
    qp[h] = g + 8 * h < TILE && R < n_rows ? q + (size_t)(u.row0 + R / G) * q_stride + (size_t)(kh * G + R % G) * D : nullptr;
  }
  Rows walk;
  walk.begin(qp, lane);

  const size_t page_stride = (size_t)HKV * KRK_PAGE * D, head_off = (size_t)kh * KRK_PAGE * D;
  auto issue = [&](int i) {  // cp.async: page i of this block's share into its stage; one group per call
    if (i < n_pages) {
      const int page = seg.table[(size_t)u.slot * seg.width + j_lo + i];
      bf16* dst = ring_s + (size_t)(i % CP_STAGES) * 2 * UNIT_ELEMS;
      load_page(dst, k_cache + (size_t)page * page_stride + head_off);
      load_page(dst + UNIT_ELEMS, v_cache + (size_t)page * page_stride + head_off);
    }
    cp_async_commit();
  };
  bool alive = true;  // false once a wait ran out: the flow stays the same for all warps, the results are void
  auto arrived = [&](int n) {
    if (alive && !tc::mbar_wait(full_bar + n % units_in_ring, (uint32_t)(n / units_in_ring) & 1)) {
      alive = false;
      if (lane == 0) atomicExch(error, 25);
    }
  };
  auto hand_back = [&](int n) {
    __syncwarp();
    if (lane == 0) tc::mbar_arrive(empty_bar + n % units_in_ring);
  };
  if (!TMA) issue(0);
  for (int i = 0; i < n_pages; ++i) {
    const int j = j_lo + i, nk = 2 * i, nv = nk + 1;
    bf16 *ks_s, *vs_s;
    if (TMA) {
      ks_s = ring_s + (size_t)(nk % units_in_ring) * UNIT_ELEMS;
      vs_s = ring_s + (size_t)(nv % units_in_ring) * UNIT_ELEMS;
      arrived(nk);
    } else {
      ks_s = ring_s + (size_t)(i % CP_STAGES) * 2 * UNIT_ELEMS;
      vs_s = ks_s + UNIT_ELEMS;
      issue(i + 1);
      cp_async_wait<1>();
      __syncthreads();
    }
    const int key0 = warp * 16, count = u.key_hi - j * KRK_PAGE;  // keys of the page that count
    walk.template scores<TMA>(ks_s, key0, count, scale_log2, lane);
    if (TMA) hand_back(nk);
    if (SUMS) walk.keep_scores(ks.raw + ((size_t)blockIdx.z * HQ + kh * G) * ks.capacity + j * KRK_PAGE + key0, ks.capacity, q_rows, lane);
    walk.update(lane);
    if (TMA) arrived(nv);
    if (count < KRK_PAGE) {  // values behind the sequence's last may be anything, and zero times infinity is not zero
      for (int e = threadIdx.x; e < (KRK_PAGE - count) * (D / 8); e += 128)
        *reinterpret_cast<uint4*>(vs_s + page_off<TMA>(count + e / (D / 8), e % (D / 8))) = make_uint4(0, 0, 0, 0);
      consumer_sync();
    }
    walk.template values<TMA>(vs_s, key0, lane);
    if (TMA) hand_back(nv);
    else __syncthreads();
  }
  if (!TMA) cp_async_wait<0>();
  else if (!alive) tc::wait_for_copies(full_bar, units_in_ring, 2 * n_pages);  // the ring's place is used again
  consumer_sync();  // every warp is done with the ring: it now holds the warps' parts

  walk.leave(red + (size_t)warp * 16 * RP, lane);
  consumer_sync();
  if (clustered) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // every block of the cluster has started
  if (!PREFIX && !clustered && !wait_first) grid_dependency_wait();                    // the prefix parts are there
  float* inbox0 = clustered ? cluster.map_shared_rank(inbox, 0) : nullptr;
  const size_t part_step = (size_t)parts.rows * parts.HQ;

  // the prefix parts of a row join what the row has from its own keys, and the row is written; a warp's lanes hold its columns
  auto finish = [&](int r, float big, float total, float (&acc)[(D + 31) / 32]) {
    const int R = rt * TILE + r, head = kh * G + R % G;
    const size_t item = (size_t)(u.row0 + R / G) * HQ + head;
    if (n_join > 0) {
      float mine = big;
      for (int p = lane; p < n_join; p += 32) mine = fmaxf(mine, parts.ml[p * part_step + item].x);
      const float all = warp_max(mine), safe = all == -INFINITY ? 0.f : all;
      const float w = exp2f(big - safe);
      total *= w;
#pragma unroll
      for (int i = 0; i < (D + 31) / 32; ++i) acc[i] *= w;
      // eight parts at once: their loads are on their way together, and a part without a key has no weight and is not read
      for (int p0 = 0; p0 < n_join; p0 += 8) {
        float wp[8], v[8][(D + 31) / 32];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float2 ml = p0 + e < n_join ? parts.ml[(p0 + e) * part_step + item] : make_float2(0.f, 0.f);
          wp[e] = ml.y == 0.f ? 0.f : exp2f(ml.x - safe);
          total += ml.y == 0.f ? 0.f : wp[e] * ml.y;
#pragma unroll
          for (int i = 0; i < (D + 31) / 32; ++i) {
            const int d = lane + 32 * i;
            v[e][i] = ml.y != 0.f && d < D ? parts.o[((p0 + e) * part_step + item) * D + d] : 0.f;
          }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
          for (int i = 0; i < (D + 31) / 32; ++i) acc[i] += wp[e] * v[e][i];
      }
    }
    const float inv = 1.f / total;
#pragma unroll
    for (int i = 0; i < (D + 31) / 32; ++i) {
      const int d = lane + 32 * i;
      if (d < D) out[item * D + d] = __float2bfloat16_rn(acc[i] * inv);
    }
  };

  for (int r = warp; r < q_rows; r += 4) {  // the four warps' parts of a row, in warp order
    float mw[4], big = -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; ++w) { mw[w] = red[((size_t)w * 16 + r) * RP + D]; big = fmaxf(big, mw[w]); }
    const float safe = big == -INFINITY ? 0.f : big;
    float wgt[4], total = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) { wgt[w] = exp2f(mw[w] - safe); total += wgt[w] * red[((size_t)w * 16 + r) * RP + D + 1]; }
    float acc[(D + 31) / 32];
#pragma unroll
    for (int i = 0; i < (D + 31) / 32; ++i) {
      const int d = lane + 32 * i;
      acc[i] = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) acc[i] += d < D ? wgt[w] * red[((size_t)w * 16 + r) * RP + d] : 0.f;
    }
    if (PREFIX) {
      const int R = rt * TILE + r;
      const size_t to = parts.at(part0 + split, u.row0 + R / G, kh * G + R % G);
      if (total != 0.f)
#pragma unroll
        for (int i = 0; i < (D + 31) / 32; ++i)
          if (lane + 32 * i < D) parts.o[to * D + lane + 32 * i] = acc[i];
      if (lane == 0) parts.ml[to] = make_float2(big, total);
    } else if (clustered) {
      float* dst = inbox0 + ((size_t)split * inbox_rows + r) * RP;
#pragma unroll
      for (int i = 0; i < (D + 31) / 32; ++i)
        if (lane + 32 * i < D) dst[lane + 32 * i] = acc[i];
      if (lane == 0) { dst[D] = big; dst[D + 1] = total; }
    } else {
      finish(r, big, total, acc);
      if (SUMS && lane == 0) lse_s[r] = safe + log2f(total);
    }
  }
  if (clustered) {
    cluster.sync();  // every block's part has arrived in the first one
    if (split == 0) {
      if (!wait_first) grid_dependency_wait();
      for (int r = warp; r < q_rows; r += 4) {  // the splits' parts of a row, in split order
        const float* mine = inbox + (size_t)r * RP;
        float big = -INFINITY;
        for (int p = lane; p < n_splits; p += 32) big = fmaxf(big, mine[(size_t)p * inbox_rows * RP + D]);
        big = warp_max(big);
        const float safe = big == -INFINITY ? 0.f : big;
        float total = 0.f, acc[(D + 31) / 32];
#pragma unroll
        for (int i = 0; i < (D + 31) / 32; ++i) acc[i] = 0.f;
        for (int p = 0; p < n_splits; ++p) {
          const float* from = mine + (size_t)p * inbox_rows * RP;
          const float w = exp2f(from[D] - safe);
          total += w * from[D + 1];
#pragma unroll
          for (int i = 0; i < (D + 31) / 32; ++i)
            if (lane + 32 * i < D) acc[i] += w * from[lane + 32 * i];
        }
        finish(r, big, total, acc);
        if (SUMS) {
          const float lse = safe + log2f(total);
          for (int p = lane; p < n_splits; p += 32) cluster.map_shared_rank(lse_s, p)[r] = lse;
        }
      }
    }
    if (SUMS) cluster.sync();
  } else if (SUMS) {
    consumer_sync();
  }
  if (SUMS) {
    const int end = min(j_hi * KRK_PAGE, u.key_hi);
    const float* raw = ks.raw + ((size_t)blockIdx.z * HQ + kh * G) * ks.capacity;
    const size_t place = ((size_t)u.slot * HKV + kh) * ks.capacity;
    constexpr int AHEAD = 8;  // keys of a thread whose loads are on their way together
    for (int key0 = j_lo * KRK_PAGE + threadIdx.x; key0 < end; key0 += 128 * AHEAD) {
      float w[AHEAD], old[AHEAD];
#pragma unroll
      for (int e = 0; e < AHEAD; ++e) {
        const int key = key0 + 128 * e;
        w[e] = 0.f;
        old[e] = key < min(end, u.start) ? ks.sums[place + key] : 0.f;
      }
      for (int r = 0; r < q_rows; ++r) {
        const float* row = raw + (size_t)r * ks.capacity;
        float s[AHEAD];
#pragma unroll
        for (int e = 0; e < AHEAD; ++e) s[e] = key0 + 128 * e < end ? row[key0 + 128 * e] : -INFINITY;
#pragma unroll
        for (int e = 0; e < AHEAD; ++e) w[e] += exp2f(s[e] - lse_s[r]);
      }
#pragma unroll
      for (int e = 0; e < AHEAD; ++e) {
        const int key = key0 + 128 * e;
        if (key >= end) break;
        ks.sums_out[place + key] = old[e] + w[e];
        if (ks.positions && key >= u.start) ks.positions[place + key] = key + (ks.seq_shift ? ks.seq_shift[blockIdx.z] : 0);
      }
    }
  }
}

template <bool PREFIX, bool SUMS, typename Rows>
int launch_few_rows(bf16* out, const Parts& parts, int part0, int n_join, const void* q, int q_stride, int HQ, int HKV, const Segments& seg,
                    const void* k, const void* v, int n_pages, int max_rows, int n_splits, float scale, bool wait_first, const KeySums& ks, int* error,
                    cudaStream_t stream) {
  const int G = HQ / HKV;
  const long long row_tiles = ((long long)max_rows * G + Rows::TILE - 1) / Rows::TILE;
  const int units = PREFIX ? seg.n_groups : seg.n_seqs;
  if (row_tiles * HKV > 65535 || units > 65535) return -3;
  const int inbox_rows = G < Rows::TILE ? G : Rows::TILE;
  // A cluster's parts meet beside the ring of pages: of large heads fewer, where not all fit (pages by cp.async, which take four places: heads of 240 and
  // 14 or more of them a kv head in eight parts would take 236 KB or more).
  constexpr size_t MOST = 227 * 1024;
  if (!PREFIX)
    while (n_splits > 1 && Layout(TMA_PAGES ? 2 : 2 * CP_STAGES, n_splits, inbox_rows).total + 1024 > MOST) n_splits /= 2;
  const int splits_in_cluster = PREFIX ? 1 : n_splits;
  const long long blocks = row_tiles * HKV * units * n_splits;
  CUtensorMap map_k = {}, map_v = {};
  int in_ring;
  if (TMA_PAGES) {
    const long long rows = (long long)n_pages * HKV * KRK_PAGE;
    int rc = tc::make_map_bf16(&map_k, k, rows, D, D, KRK_PAGE);
    if (rc == 0) rc = tc::make_map_bf16(&map_v, v, rows, D, D, KRK_PAGE);
    if (rc) return rc;
    // As many units as the shared memory of an SM holds for the blocks that it gets. Clusters of four or eight do not fill every SM: 33 and 15 of them
    // run at once with a block an SM, and more wait for a second
    // round: 16 sequences' kv heads in clusters of eight after 1,500 keys 17.5 us by the device's 148 and 10.0 by 120, 36 in clusters of four 21.9 and 12.9.
    const int fit = splits_in_cluster >= 8 ? 120 : splits_in_cluster >= 4 ? 132 : 148;
    const int per_sm = blocks <= fit ? 1 : blocks <= 2 * fit ? 2 : blocks <= 3 * fit || Rows::TILE == 16 ? 3 : 4;
    const size_t room = 216 * 1024 / per_sm, fixed = Layout(0, splits_in_cluster, inbox_rows).total - Layout(0, 1, 0).total + 2048;
    in_ring = (int)((room > fixed ? room - fixed : 0) / UNIT_BYTES);
    in_ring = in_ring < 2 ? 2 : in_ring > 12 ? 12 : in_ring;
  } else {
    in_ring = 2 * CP_STAGES;
  }
  const size_t smem = Layout(in_ring, splits_in_cluster, inbox_rows).total + 1024;
  if (smem > MOST) return -2;
  auto kern = few_rows_kernel<TMA_PAGES, PREFIX, SUMS, Rows>;
  static unsigned long long allowed = 0;
  cudaError_t e = allow_shared(kern, MOST, &allowed);
  if (e != cudaSuccess) return (int)e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)n_splits, (unsigned)(row_tiles * HKV), (unsigned)units);
  cfg.blockDim = dim3(TMA_PAGES ? 160 : 128);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = splits_in_cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return (int)cudaLaunchKernelEx(&cfg, kern, map_k, map_v, out, parts, part0, n_join, (const bf16*)q, q_stride, HQ, HKV, seg, (const bf16*)k,
                                 (const bf16*)v, scale * LOG2E, (int)row_tiles, in_ring, wait_first, ks, error);
}

}  // namespace

#define KRK_SEGMENTS                                                                                                                    \
  const int *cu_q, const int *seq_slot, const int *seq_start, const int *seq_qlen, const int *group_cu, const int *group_len,             \
      const int *seq_group, int n_seqs, int n_groups, const int *table, int width
#define KRK_MAKE_SEGMENTS \
  Segments { cu_q, seq_slot, seq_start, seq_qlen, group_cu, group_len, seq_group, n_seqs, n_groups, table, width }

// Parts part0 .. part0 + n_splits - 1 of the groups' prefixes; max_rows: the most rows of the step that a group has.
KRK_API int krk_prefix_few_rows(float* o, float* ml, int rows, int part0, int n_splits, const void* q, int q_stride, int HQ, int HKV, KRK_SEGMENTS,
                                const void* k_cache, const void* v_cache, int n_pages, int max_rows, float scale, int* error, cudaStream_t stream) {
  if (rows == 0 || n_groups == 0) return 0;
  const Parts parts = {o, (float2*)ml, rows, HQ};
  auto go = (long long)max_rows * (HQ / HKV) <= 8 ? launch_few_rows<true, false, Narrow> : launch_few_rows<true, false, Wide>;
  return go(nullptr, parts, part0, 0, q, q_stride, HQ, HKV, KRK_MAKE_SEGMENTS, k_cache, v_cache, n_pages, max_rows, n_splits, scale, true, KeySums{}, error,
            stream);
}

// One token a sequence: its own keys (all, without groups), joined with the prefix parts 0 .. n_join - 1, which the launch before this one
// writes (n_join 0: none, and the launch before may write the rows and keys themselves). n_splits: at most 8, blocks of a cluster.
static int krk_own_single(void* out, const float* o, const float* ml, int n_join, int n_splits, const void* q, int q_stride, int HQ, int HKV,
                           KRK_SEGMENTS, const void* k_cache, const void* v_cache, int n_pages, float scale, int* error, cudaStream_t stream) {
  if (n_seqs == 0) return 0;
  const Parts parts = {const_cast<float*>(o), (float2*)const_cast<float*>(ml), n_seqs, HQ};
  auto go = HQ / HKV <= 8 ? launch_few_rows<false, false, Narrow> : launch_few_rows<false, false, Wide>;
  return go((bf16*)out, parts, 0, n_join, q, q_stride, HQ, HKV, KRK_MAKE_SEGMENTS, k_cache, v_cache, n_pages, 1, n_splits, scale, n_join == 0, KeySums{},
            error, stream);
}

extern "C" int krk_prefix_tcgen05(float*, float*, int, int, int, const void*, int, int, int, const int*, const int*, const int*, const int*, const int*,
                                  const int*, const int*, int, int, const int*, int, const void*, const void*, int, int, int, float, int*, cudaStream_t);

// A single-token step behind shared prefixes, both launches: n_splits parts of the prefixes (none: 0; `tensor` 1: by the tcgen05 kernel, 2: by its
// halves, n_splits each), then the own keys, shared by own_splits blocks a sequence, which join them. o, ml: scratch for the parts of n_seqs rows.
KRK_API int krk_shared_single(void* out, float* o, float* ml, int n_splits, int own_splits, int tensor, const void* q, int q_stride, int HQ, int HKV,
                              KRK_SEGMENTS, const void* k_cache, const void* v_cache, int n_pages, int max_rows, float scale, int* error,
                              cudaStream_t stream) {
  if (n_splits > 0) {
    int rc;
#if KRK_HEAD_DIM == 64 || KRK_HEAD_DIM == 128
    if (tensor)
      rc = krk_prefix_tcgen05(o, ml, n_seqs, 0, n_splits, q, q_stride, HQ, HKV, cu_q, seq_slot, seq_start, seq_qlen, group_cu, group_len, seq_group, n_seqs,
                              n_groups, table, width, k_cache, v_cache, n_pages, max_rows, tensor == 2, scale, error, stream);
    else
#endif
      rc = krk_prefix_few_rows(o, ml, n_seqs, 0, n_splits, q, q_stride, HQ, HKV, cu_q, seq_slot, seq_start, seq_qlen, group_cu, group_len, seq_group, n_seqs,
                               n_groups, table, width, k_cache, v_cache, n_pages, max_rows, scale, error, stream);
    if (rc) return rc;
  }
  return krk_own_single(out, o, ml, tensor == 2 ? 2 * n_splits : n_splits, own_splits, q, q_stride, HQ, HKV, cu_q, seq_slot, seq_start, seq_qlen, group_cu, group_len, seq_group, n_seqs,
                        n_groups, table, width, k_cache, v_cache, n_pages, scale, error, stream);
}

// One token a sequence over all of its keys, with the weight that each key receives added to its sum (see krk_key_weights). raw: scratch,
// [n_seqs][HQ][capacity]. The heads of a kv head fit one tile: HQ / HKV <= 16 (-2 otherwise).
KRK_API int krk_scored_single(void* out, float* raw, const float* sums, float* sums_out, int* positions, const int* seq_shift, int capacity,
                              int n_splits, const void* q, int q_stride, int HQ, int HKV, KRK_SEGMENTS, const void* k_cache, const void* v_cache,
                              int n_pages, float scale, int* error, cudaStream_t stream) {
  if (n_seqs == 0) return 0;
  if (HQ / HKV > 16) return -2;
  auto go = HQ / HKV <= 8 ? launch_few_rows<false, true, Narrow> : launch_few_rows<false, true, Wide>;
  return go((bf16*)out, Parts{nullptr, nullptr, n_seqs, HQ}, 0, 0, q, q_stride, HQ, HKV, KRK_MAKE_SEGMENTS, k_cache, v_cache, n_pages, 1, n_splits, scale, true,
            KeySums{raw, sums, sums_out, positions, seq_shift, capacity}, error, stream);
}

#endif  // head sizes served by these kernels
