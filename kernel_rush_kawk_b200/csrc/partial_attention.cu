// Attention in parts over the paged cache with ordinary arithmetic, for every type and head size: the parts of a shared
// prefix and of a sequence's own keys, their join, and the weight that each key received. See partial_attention.cuh for what
// the parts are.
//
// A block takes TILE (token, head) rows of one kv head and walks pages of 64 keys, brought to shared memory as float32. Thread (ty, tx) of
// 16 x 16 has rows ty + 16 i and keys tx + 16 j of S = Q K^T, four by four in registers, and columns 4 tx + 64 c of the same rows of O: a row's
// statistics and its weights stay within half a warp. Weights stay float32. A product of 64 multiply-adds a thread reads 8 pieces of 16 bytes,
// 12 shared-memory wavefronts a warp in the 16 clocks that the multiply-adds take. Tiles of fewer rows skip the places behind them by sixteens.
//
// What bounds it, float32: of single tokens the dependent steps of two or three launches (six sequences behind 960 positions, 16 heads over 4 of 64: 11.3 us for
// the parts; 15 in tiles of 16 rows by 128 threads, the form before this one); of many rows issue slots and latencies at 16 warps an SM: two sequences of 300
// tokens behind 512 positions, 32 heads over 8 of 128: 269 us, 23 TFLOP/s of 72 (430 in tiles of 16). Eight rows a thread by 128 threads
// (fewer reads, fewer warps) took 335, three blocks an SM in 80 registers spilled and gained nothing.
//
// Compiled once per head size: -DKRK_HEAD_DIM=<D>.
#include "mma.cuh"
#include "partial_attention.cuh"
#include "tcgen05.cuh"

#ifndef KRK_HEAD_DIM
#error "compile with -DKRK_HEAD_DIM=<head size>"
#endif

namespace {

constexpr int D = KRK_HEAD_DIM;
constexpr int DPAD = (D + 3) / 4 * 4;  // columns in shared memory; those behind D are zero
constexpr int PITCH = DPAD / 4 % 2 ? DPAD : DPAD + 4;  // floats between rows of queries and keys: eight neighbouring rows' pieces fall into different banks
constexpr int P_PITCH = KRK_PAGE + 4;
constexpr int TILE = 64;               // rows of a block
constexpr int THREADS = 256;
constexpr int JOIN_THREADS = 128;
constexpr int MAX_SHARE = 8;           // blocks of a cluster that share a page's row tiles
constexpr int CHUNKS = (DPAD + 63) / 64;  // of columns: a thread has four of each
constexpr int PER_LANE = (D + 31) / 32;
constexpr float LOG2E = 1.4426950408889634f;
// Where the head is large the weights lie where the keys were, so that two blocks fit an SM; it costs a barrier a page.
constexpr bool OVER_KEYS = D > 64;

struct Shared {
  float q[TILE * PITCH];
  float k[KRK_PAGE * PITCH];
  float v[KRK_PAGE * PITCH];  // [key][DPAD]; of the weights' kernel a second tile of queries
  float p[OVER_KEYS ? 4 : TILE * P_PITCH];  // weights, [row][key]
};
static_assert(!OVER_KEYS || PITCH >= P_PITCH, "");
constexpr size_t SMEM_BYTES = sizeof(Shared);

// 64 rows of D elements, row r from row(r) on, as float32; rows from `count` (1 or more) on become zero, so that what they hold counts nowhere. `pieces`: every row
// starts on a 16-byte boundary. Rows of float32 are on their way when the call returns (cp.async; a group of its own), others are there.
template <typename T, int STRIDE, typename Row>
__device__ __forceinline__ void load_tile(float* dst, int count, bool pieces, Row row) {
  constexpr int V = 16 / sizeof(T);  // elements of a 16-byte piece
  if (sizeof(T) == 4 && D % V == 0 && pieces) {
    for (int i = threadIdx.x; i < 64 * (D / V); i += THREADS) {
      const int r = i / (D / V), c = i % (D / V) * V;
      const uint32_t to = (uint32_t)__cvta_generic_to_shared(dst + r * STRIDE + c);
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(row(min(r, count - 1)) + c), "r"(r < count ? 16 : 0) : "memory");
    }
    cp_async_commit();
    return;
  }
  cp_async_commit();  // (an empty group: the waits count groups)
  if (D % V == 0 && pieces) {
    constexpr int ALL = 64 * (D / V), AHEAD = 4;  // a thread's pieces four at a time, so that their loads are on their way together
    for (int i0 = threadIdx.x; i0 < ALL; i0 += THREADS * AHEAD) {
      uint4 x[AHEAD];
#pragma unroll
      for (int a = 0; a < AHEAD; ++a) {
        const int i = i0 + a * THREADS, r = i / (D / V);
        x[a] = i < ALL && r < count ? *reinterpret_cast<const uint4*>(row(r) + i % (D / V) * V) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int a = 0; a < AHEAD; ++a) {
        const int i = i0 + a * THREADS;
        if (i >= ALL) break;
        const T* e = reinterpret_cast<const T*>(x + a);
        float* to = dst + i / (D / V) * STRIDE + i % (D / V) * V;
#pragma unroll
        for (int c = 0; c < V; c += 4) *reinterpret_cast<float4*>(to + c) = make_float4(to_float<T>(e[c]), to_float<T>(e[c + 1]), to_float<T>(e[c + 2]), to_float<T>(e[c + 3]));
      }
    }
    return;
  }
  for (int i = threadIdx.x; i < 64 * DPAD; i += THREADS) {
    const int r = i / DPAD, d = i % DPAD;
    dst[r * STRIDE + d] = r < count && d < D ? to_float<T>(row(r)[d]) : 0.f;
  }
}

// Rows `tile` of one kv head's n_rows (token, head) rows from row0 on.
template <typename T>
__device__ __forceinline__ void load_queries(float* dst, const T* __restrict__ q, int q_stride, int row0, int n_rows, int tile, int G, int kh) {
  const bool pieces = (((uintptr_t)q | (q_stride * sizeof(T)) | (D * sizeof(T))) & 15) == 0;
  load_tile<T, PITCH>(dst, n_rows - tile * TILE, pieces, [&](int r) {
    const int R = tile * TILE + r;
    return q + (size_t)(row0 + R / G) * q_stride + (size_t)(kh * G + R % G) * D;
  });
}

template <typename T, int STRIDE>
__device__ __forceinline__ void load_page(float* dst, const T* __restrict__ page, int count) {
  load_tile<T, STRIDE>(dst, count, ((uintptr_t)page & 15) == 0, [&](int r) { return page + r * D; });
}

// Scores of rows ty + 16 i (i below `live`) with keys tx + 16 j.
__device__ __forceinline__ void scores(const float* q_s, const float* k_s, int live, float (&s)[4][4]) {
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) s[i][j] = 0.f;
#pragma unroll 2
  for (int d = 0; d < DPAD; d += 4) {
    float4 k[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) k[j] = *reinterpret_cast<const float4*>(k_s + (tx + 16 * j) * PITCH + d);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i >= live) break;
      const float4 q = *reinterpret_cast<const float4*>(q_s + (ty + 16 * i) * PITCH + d);
#pragma unroll
      for (int j = 0; j < 4; ++j) s[i][j] = fmaf(k[j].x, q.x, fmaf(k[j].y, q.y, fmaf(k[j].z, q.z, fmaf(k[j].w, q.w, s[i][j]))));
    }
  }
}

// Block (tile x split, kv head, group or sequence): the groups' prefixes first, in n_prefix parts, then the sequences' own keys in
// n_own more.
template <typename T>
__global__ void __launch_bounds__(THREADS, D <= 128 ? 2 : 1)
partial_attention_kernel(Parts parts, int n_prefix, int n_own, const T* __restrict__ q, int q_stride, int HQ, int HKV, Segments seg,
                         const T* __restrict__ k_cache, const T* __restrict__ v_cache, float scale_log2) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  Shared& sm = *reinterpret_cast<Shared*>(smem_raw);
  grid_dependency_wait();
  grid_launch_dependents();  // in this order: the kernel behind a prefix's parts reads rows and keys before it waits for these
  const int kh = blockIdx.y, G = HQ / HKV;
  const int groups = n_prefix > 0 ? seg.n_groups : 0;
  const bool own = (int)blockIdx.z >= groups;
  const int n_splits = own ? n_own : n_prefix, part0 = own ? n_prefix : 0;
  const int split = blockIdx.x % n_splits, tile = blockIdx.x / n_splits;
  const Unit u = own ? own_unit(seg, blockIdx.z - groups) : prefix_unit(seg, blockIdx.z);
  const int n_rows = u.n_tok * G;
  if (tile * TILE >= n_rows) return;
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  const int live = min(4, (n_rows - tile * TILE + 15) / 16);
  const int last_tok = min(u.n_tok - 1, (tile * TILE + TILE - 1) / G);
  const int key_end = own ? min(u.key_hi, u.start + last_tok + 1) : u.key_hi;  // behind the last key that the tile sees
  int j_lo, j_hi;
  split_pages(u.key_lo, key_end, split, n_splits, j_lo, j_hi);

  auto load_k = [&](int j) {
    const size_t page = (size_t)seg.table[(size_t)u.slot * seg.width + j] * HKV + kh;
    load_page<T, PITCH>(sm.k, k_cache + page * KRK_PAGE * D, min(KRK_PAGE, key_end - j * KRK_PAGE));
  };
  auto load_v = [&](int j) {
    const size_t page = (size_t)seg.table[(size_t)u.slot * seg.width + j] * HKV + kh;
    load_page<T, DPAD>(sm.v, v_cache + page * KRK_PAGE * D, min(KRK_PAGE, key_end - j * KRK_PAGE));
  };
  if (j_lo < j_hi) {
    load_queries(sm.q, q, q_stride, u.row0, n_rows, tile, G, kh);
    load_k(j_lo);
    load_v(j_lo);
  }
  float m[4], l[4], acc[4][CHUNKS][4];  // l: of this thread's keys alone, until the end
  int row_end[4];                       // behind the last key that the row sees
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
    row_end[i] = min(key_end, u.start + (tile * TILE + ty + 16 * i) / G + 1);
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][c][e] = 0.f;
  }
  float* p_s = OVER_KEYS ? sm.k : sm.p;

  for (int j = j_lo; j < j_hi; ++j) {
    const int key0 = j * KRK_PAGE, count = min(KRK_PAGE, key_end - key0);
    cp_async_wait<1>();
    __syncthreads();  // the keys are here
    float s[4][4];
    scores(sm.q, sm.k, live, s);
    cp_async_wait<0>();
    __syncthreads();  // the values are here, and the keys' place is free
    if (!OVER_KEYS && j + 1 < j_hi) load_k(j + 1);
    const bool whole = key0 + KRK_PAGE <= min(key_end, u.start + tile * TILE / G + 1);  // every row sees the page to its end
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i >= live) break;
      const int seen = row_end[i] - key0;  // keys of the page that the row sees
      float mx = -INFINITY;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[i][e] = tx + 16 * e < seen ? s[i][e] * scale_log2 : -INFINITY;
        mx = fmaxf(mx, s[i][e]);
      }
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      const float m_new = fmaxf(m[i], mx), safe = m_new == -INFINITY ? 0.f : m_new, alpha = exp2f(m[i] - safe);
      m[i] = m_new;
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float p = exp2f(s[i][e] - safe);
        if (tx + 16 * e < seen) sum += p;
        p_s[(ty + 16 * i) * P_PITCH + tx + 16 * e] = tx + 16 * e < seen ? p : -1.f;  // no weight: what the value is does not count
      }
      l[i] = l[i] * alpha + sum;
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][c][e] *= alpha;
    }
    __syncwarp();  // a row's weights come from the half warp that reads them
    if (whole) {
#pragma unroll 2
      for (int key = 0; key < KRK_PAGE; key += 4) {
        float4 p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i < live) p[i] = *reinterpret_cast<const float4*>(p_s + (ty + 16 * i) * P_PITCH + key);
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
          const int d = 4 * tx + 64 * c;
          if (DPAD % 64 && d >= DPAD) break;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float4 v = *reinterpret_cast<const float4*>(sm.v + (key + e) * DPAD + d);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if (i >= live) break;
              const float w = e == 0 ? p[i].x : e == 1 ? p[i].y : e == 2 ? p[i].z : p[i].w;
              acc[i][c][0] = fmaf(w, v.x, acc[i][c][0]);
              acc[i][c][1] = fmaf(w, v.y, acc[i][c][1]);
              acc[i][c][2] = fmaf(w, v.z, acc[i][c][2]);
              acc[i][c][3] = fmaf(w, v.w, acc[i][c][3]);
            }
          }
        }
      }
    } else {
      for (int key = 0; key < count; ++key) {
        float p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = i < live ? p_s[(ty + 16 * i) * P_PITCH + key] : -1.f;
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
          const int d = 4 * tx + 64 * c;
          if (DPAD % 64 && d >= DPAD) break;
          const float4 v = *reinterpret_cast<const float4*>(sm.v + key * DPAD + d);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (p[i] >= 0.f || p[i] != p[i]) {
              acc[i][c][0] = fmaf(p[i], v.x, acc[i][c][0]);
              acc[i][c][1] = fmaf(p[i], v.y, acc[i][c][1]);
              acc[i][c][2] = fmaf(p[i], v.z, acc[i][c][2]);
              acc[i][c][3] = fmaf(p[i], v.w, acc[i][c][3]);
            }
        }
      }
    }
    if (j + 1 < j_hi) {
      __syncthreads();  // the values have been read
      if (OVER_KEYS) load_k(j + 1);
      load_v(j + 1);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (i >= live) break;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], o);
    const int R = tile * TILE + ty + 16 * i;
    if (R >= n_rows) continue;
    const size_t at = parts.at(part0 + split, u.row0 + R / G, kh * G + R % G);
    if (l[i] != 0.f)  // (a NaN is none)
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (4 * tx + 64 * c + e < D) parts.o[at * D + 4 * tx + 64 * c + e] = acc[i][c][e];
    if (tx == 0) parts.ml[at] = make_float2(m[i], l[i]);
  }
}

// One warp per (row, head): the parts' join. lse (may be null): log2 of the sum of the row's 2^s, for the weights of its keys.
template <typename T>
__global__ void __launch_bounds__(JOIN_THREADS) join_parts_kernel(T* __restrict__ out, float* __restrict__ lse, Parts parts, int n_parts) {
  grid_launch_dependents();
  grid_dependency_wait();
  const long long item = (long long)blockIdx.x * (JOIN_THREADS / 32) + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (item >= (long long)parts.rows * parts.HQ) return;
  const size_t step = (size_t)parts.rows * parts.HQ;
  float big = -INFINITY, total = 0.f;
  float acc[PER_LANE];
#pragma unroll
  for (int i = 0; i < PER_LANE; ++i) acc[i] = 0.f;
  for (int p = lane; p < n_parts; p += 32) big = fmaxf(big, parts.ml[p * step + item].x);
  big = warp_max(big);
  const float safe = big == -INFINITY ? 0.f : big;
  constexpr int AHEAD = PER_LANE <= 4 ? 8 : 4;  // parts whose loads are on their way together
  for (int p0 = 0; p0 < n_parts; p0 += AHEAD) {
    float w[AHEAD], v[AHEAD][PER_LANE];
#pragma unroll
    for (int e = 0; e < AHEAD; ++e) {
      const float2 ml = p0 + e < n_parts ? parts.ml[(p0 + e) * step + item] : make_float2(0.f, 0.f);
      w[e] = ml.y == 0.f ? 0.f : exp2f(ml.x - safe);
      total += ml.y == 0.f ? 0.f : w[e] * ml.y;
#pragma unroll
      for (int i = 0; i < PER_LANE; ++i) {
        const int d = lane + 32 * i;
        v[e][i] = ml.y != 0.f && d < D ? parts.o[((p0 + e) * step + item) * D + d] : 0.f;
      }
    }
#pragma unroll
    for (int e = 0; e < AHEAD; ++e)
#pragma unroll
      for (int i = 0; i < PER_LANE; ++i) acc[i] += w[e] * v[e][i];
  }
  const float inv = 1.f / total;
#pragma unroll
  for (int i = 0; i < PER_LANE; ++i) {
    const int d = lane + 32 * i;
    if (d < D) out[item * D + d] = from_float<T>(acc[i] * inv);
  }
  if (lse && lane == 0) lse[item] = safe + log2f(total);
}

// The weight that each key of a sequence receives from the step's last `observe` queries (all of them where it is 0), added up
// over the heads of its kv head: sums_out = sums + weight for keys held before the step, the weight alone for the step's
// own. Block (pages x, x + gridDim.x / share, ..., kv head, sequence); a cluster's `share` blocks take the row tiles of a page in turn, and the first adds
// their sums up in order.
template <typename T>
__global__ void __launch_bounds__(THREADS, D <= 128 ? 2 : 1)
key_weights_kernel(const float* sums, float* sums_out, int* __restrict__ positions, const int* __restrict__ seq_shift, int capacity,
                   const float* __restrict__ lse, int observe, const T* __restrict__ q, int q_stride, int HQ, int HKV, Segments seg,
                   const T* __restrict__ k_cache, float scale_log2, int share) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  Shared& sm = *reinterpret_cast<Shared*>(smem_raw);
  __shared__ float minus_lse[2][TILE], warp_sums[THREADS / 32][KRK_PAGE], inbox[MAX_SHARE][KRK_PAGE];
  if (share > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // "I have started"
  grid_launch_dependents();
  grid_dependency_wait();
  if (share > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  const int rank = blockIdx.x % share, kh = blockIdx.y, seq = blockIdx.z, G = HQ / HKV;
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Unit u = own_unit(seg, seq);
  const int seen = observe > 0 ? min(observe, u.n_tok) : u.n_tok, tok0 = u.n_tok - seen;
  const int n_rows = seen * G, row0 = u.row0 + tok0, start = u.start + tok0;
  for (int j = blockIdx.x / share; j * KRK_PAGE < u.key_hi; j += gridDim.x / share) {
    const int page = seg.table[(size_t)u.slot * seg.width + j], key0 = j * KRK_PAGE;
    const size_t base = ((size_t)page * HKV + kh) * KRK_PAGE * D;
    __syncthreads();  // the sums of the page before have been read
    load_page<T, PITCH>(sm.k, k_cache + base, min(KRK_PAGE, u.key_hi - key0));
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
    const int first = max(0, key0 - start) * G / TILE + rank;  // of the tiles with a row that sees the page's first key, this block's first
    auto load = [&](int tile, int place) {
      load_queries(place ? sm.v : sm.q, q, q_stride, row0, n_rows, tile, G, kh);
      if (threadIdx.x < TILE) {
        const int R = tile * TILE + threadIdx.x;
        minus_lse[place][threadIdx.x] = R < n_rows ? -lse[(size_t)(row0 + R / G) * HQ + kh * G + R % G] : 0.f;
      }
    };
    if (first * TILE < n_rows) load(first, 0);
    for (int tile = first, place = 0; tile * TILE < n_rows; tile += share, place ^= 1) {
      const int live = min(4, (n_rows - tile * TILE + 15) / 16);
      if ((tile + share) * TILE < n_rows) {
        load(tile + share, place ^ 1);
        cp_async_wait<1>();
      } else {
        cp_async_wait<0>();
      }
      __syncthreads();
      float s[4][4];
      scores(place ? sm.v : sm.q, sm.k, live, s);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (i >= live) break;
        const int R = tile * TILE + ty + 16 * i, end = R < n_rows ? start + R / G + 1 - key0 : 0;  // behind the last key of the page that the row sees
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (tx + 16 * e < end) sum[e] += exp2f(fmaf(s[i][e], scale_log2, minus_lse[place][ty + 16 * i]));
      }
      __syncthreads();  // the tile has been read
    }
    cp_async_wait<0>();  // of a page that no tile of this block's sees the keys are still on their way
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      sum[e] += __shfl_xor_sync(0xffffffffu, sum[e], 16);
      if (lane < 16) warp_sums[warp][tx + 16 * e] = sum[e];
    }
    __syncthreads();
    float total = 0.f;
    if (threadIdx.x < KRK_PAGE)
#pragma unroll
      for (int w = 0; w < THREADS / 32; ++w) total += warp_sums[w][threadIdx.x];
    if (share > 1) {
      if (threadIdx.x < KRK_PAGE)
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(tc::cluster_address(&inbox[rank][threadIdx.x], 0)), "f"(total) : "memory");
      tc::cluster_sync();
      total = 0.f;
      if (rank == 0 && threadIdx.x < KRK_PAGE)
        for (int c = 0; c < share; ++c) total += inbox[c][threadIdx.x];
    }
    const int at = key0 + threadIdx.x;
    if (rank == 0 && threadIdx.x < KRK_PAGE && at < u.key_hi) {
      const size_t place = ((size_t)u.slot * HKV + kh) * capacity + at;
      sums_out[place] = at < u.start ? sums[place] + total : total;
      if (positions && at >= u.start) positions[place] = at + (seq_shift ? seq_shift[seq] : 0);
    }
    if (share > 1) tc::cluster_sync();  // the first block has read what the others sent
  }
}

template <typename T>
int launch_partial(const Parts& parts, int n_prefix, int n_own, const void* q, int q_stride, int HQ, int HKV, const Segments& seg, const void* k,
                   const void* v, int group_rows, int own_rows, float scale, cudaStream_t stream) {
  auto blocks_of = [&](int rows, int splits) { return ((long long)rows * (HQ / HKV) + TILE - 1) / TILE * splits; };
  const long long prefix_blocks = n_prefix > 0 ? blocks_of(group_rows, n_prefix) : 0, own_blocks = blocks_of(own_rows, n_own);
  const long long blocks = prefix_blocks > own_blocks ? prefix_blocks : own_blocks;
  const int units = seg.n_seqs + (n_prefix > 0 ? seg.n_groups : 0);
  if (blocks > 0x7fffffffLL || HKV > 65535 || units > 65535) return -3;
  auto kern = partial_attention_kernel<T>;
  static unsigned long long allowed = 0;  // of this instance, one for each type
  cudaError_t e = allow_shared(kern, SMEM_BYTES, &allowed);
  if (e != cudaSuccess) return (int)e;
  return (int)launch_pdl(kern, dim3((unsigned)blocks, HKV, units), dim3(THREADS), SMEM_BYTES, stream, parts, n_prefix, n_own, (const T*)q, q_stride, HQ, HKV, seg, (const T*)k, (const T*)v, scale * LOG2E);
}

}  // namespace

#define KRK_SEGMENTS                                                                                                                    \
  const int *cu_q, const int *seq_slot, const int *seq_start, const int *seq_qlen, const int *group_cu, const int *group_len,             \
      const int *seq_group, int n_seqs, int n_groups, const int *table, int width
#define KRK_MAKE_SEGMENTS \
  Segments { cu_q, seq_slot, seq_start, seq_qlen, group_cu, group_len, seq_group, n_seqs, n_groups, table, width }

// Parts 0 .. n_prefix - 1 of the groups' prefixes (none: 0) and the next n_own of the sequences' other keys. group_rows, own_rows: the most rows of the
// step that a group and a sequence have.
static int krk_partial_attention(float* o, float* ml, int rows, int n_prefix, int n_own, const void* q, int q_stride, int HQ, int HKV, KRK_SEGMENTS,
                                  const void* k_cache, const void* v_cache, int group_rows, int own_rows, float scale, int dtype, cudaStream_t stream) {
  const Parts parts = {o, (float2*)ml, rows, HQ};
  const Segments seg = KRK_MAKE_SEGMENTS;
  if (rows == 0 || own_rows == 0 || n_seqs == 0 || n_own < 1) return 0;
  return dtype == KRK_DTYPE_F32 ? launch_partial<float>(parts, n_prefix, n_own, q, q_stride, HQ, HKV, seg, k_cache, v_cache, group_rows, own_rows, scale, stream)
                                : launch_partial<bf16>(parts, n_prefix, n_own, q, q_stride, HQ, HKV, seg, k_cache, v_cache, group_rows, own_rows, scale, stream);
}

static int krk_join_parts(void* out, float* lse, const float* o, const float* ml, int rows, int HQ, int n_parts, int dtype, cudaStream_t stream) {
  const Parts parts = {const_cast<float*>(o), (float2*)const_cast<float*>(ml), rows, HQ};
  const long long blocks = ((long long)rows * HQ + JOIN_THREADS / 32 - 1) / (JOIN_THREADS / 32);
  if (blocks == 0) return 0;
  if (blocks > 0x7fffffffLL) return -3;
  if (dtype == KRK_DTYPE_F32)
    return (int)launch_pdl(join_parts_kernel<float>, dim3((unsigned)blocks), dim3(JOIN_THREADS), 0, stream, (float*)out, lse, parts, n_parts);
  return (int)launch_pdl(join_parts_kernel<bf16>, dim3((unsigned)blocks), dim3(JOIN_THREADS), 0, stream, (bf16*)out, lse, parts, n_parts);
}

// page_blocks: blocks, or clusters, that share a sequence's pages; any number is right. max_seen: the most queries of a sequence that count.
KRK_API int krk_key_weights(const float* sums, float* sums_out, int* positions, const int* seq_shift, int capacity, const float* lse, int observe,
                            const void* q, int q_stride, int HQ, int HKV, KRK_SEGMENTS, const void* k_cache, int page_blocks, int max_seen, float scale,
                            int dtype, cudaStream_t stream) {
  const Segments seg = KRK_MAKE_SEGMENTS;
  if (n_seqs == 0) return 0;
  if (HKV > 65535 || n_seqs > 65535 || page_blocks < 1) return -3;
  // a page's row tiles are shared out while blocks are few for the device and each has two tiles or more
  const long long tiles = ((long long)max_seen * (HQ / HKV) + TILE - 1) / TILE, blocks = (long long)page_blocks * HKV * n_seqs;
  int share = 1;
  while (share < MAX_SHARE && blocks * share < 296 && tiles >= 4 * share) share *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)page_blocks * share, HKV, n_seqs);
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
  static unsigned long long allowed[2] = {0, 0};
  auto go = [&](auto* kern, auto* queries, auto* keys) {
    cudaError_t e = allow_shared(kern, SMEM_BYTES, allowed + (dtype == KRK_DTYPE_F32));
    if (e != cudaSuccess) return (int)e;
    return (int)cudaLaunchKernelEx(&cfg, kern, sums, sums_out, positions, seq_shift, capacity, lse, observe, queries, q_stride, HQ, HKV, seg, keys,
                                   scale * LOG2E, share);
  };
  if (dtype == KRK_DTYPE_F32) return go(key_weights_kernel<float>, (const float*)q, (const float*)k_cache);
  return go(key_weights_kernel<bf16>, (const bf16*)q, (const bf16*)k_cache);
}

// Attention in parts and their join (out; lse may be null) and, where sums_out is given, the weights of the keys, with lse as their logarithms: krk_partial_attention,
// krk_join_parts and krk_key_weights in one call. o, ml: scratch for n_prefix + n_own parts.
KRK_API int krk_attention_in_parts(void* out, float* lse, float* o, float* ml, int rows, int n_prefix, int n_own, const float* sums, float* sums_out,
                                   int* positions, const int* seq_shift, int capacity, int observe, int page_blocks, int max_seen, const void* q, int q_stride, int HQ,
                                   int HKV, KRK_SEGMENTS, const void* k_cache, const void* v_cache, int group_rows, int own_rows, float scale, int dtype,
                                   cudaStream_t stream) {
  int rc = krk_partial_attention(o, ml, rows, n_prefix, n_own, q, q_stride, HQ, HKV, cu_q, seq_slot, seq_start, seq_qlen, group_cu, group_len, seq_group,
                                 n_seqs, n_groups, table, width, k_cache, v_cache, group_rows, own_rows, scale, dtype, stream);
  if (rc == 0) rc = krk_join_parts(out, lse, o, ml, rows, HQ, n_prefix + n_own, dtype, stream);
  if (rc == 0 && sums_out)
    rc = krk_key_weights(sums, sums_out, positions, seq_shift, capacity, lse, observe, q, q_stride, HQ, HKV, cu_q, seq_slot, seq_start, seq_qlen, group_cu,
                         group_len, seq_group, n_seqs, n_groups, table, width, k_cache, page_blocks, max_seen, scale, dtype, stream);
  return rc;
}
