// Attention in parts over the paged cache with ordinary arithmetic, for every type and head size: the parts of a shared
// prefix and of a sequence's own keys, their join, and the weight that each key received. See partial_attention.cuh for what
// the parts are.
//
// A block takes TILE (token, head) rows of one kv head and walks pages of 64 keys, brought to shared memory as float32:
// S = Q K^T with a key and half the rows a thread, running maximum and sum of a row by eight threads, O += P V with a warp per
// 16 keys of the page and a lane per column; the four warps' sums of O join at the end. Weights stay float32. All rows of a tile
// share one read of K and V: with 16 rows the products take 3 shared-memory wavefronts per 8 multiply-adds a warp, two thirds
// of the multiply-add rate.
//
// Compiled once per head size: -DKRK_HEAD_DIM=<D>.
#include "partial_attention.cuh"

#ifndef KRK_HEAD_DIM
#error "compile with -DKRK_HEAD_DIM=<head size>"
#endif

namespace {

constexpr int D = KRK_HEAD_DIM;
constexpr int DPAD = (D + 3) / 4 * 4;  // columns in shared memory; those behind D are zero
constexpr int PITCH = DPAD + 4;        // floats between rows of keys: eight neighbouring keys' pieces fall into different banks
constexpr int TILE = 16;               // rows of a block
constexpr int THREADS = 128;
constexpr int PER_LANE = (D + 31) / 32;
constexpr float LOG2E = 1.4426950408889634f;

struct Shared {
  float q[TILE][DPAD];
  float k[KRK_PAGE][PITCH];
  float v[KRK_PAGE][DPAD];
  float s[KRK_PAGE][TILE + 4];  // scores, then weights, by key
  float alpha[TILE], m[TILE], l[TILE];
};
constexpr size_t SMEM_BYTES = sizeof(Shared);

template <typename T>
__device__ __forceinline__ void load_queries(Shared& sm, const T* __restrict__ q, int q_stride, int row0, int n_rows, int tile, int G, int kh) {
  for (int i = threadIdx.x; i < TILE * DPAD; i += THREADS) {
    const int r = i / DPAD, d = i % DPAD, R = tile * TILE + r;
    sm.q[r][d] = R < n_rows && d < D ? to_float<T>(q[(size_t)(row0 + R / G) * q_stride + (size_t)(kh * G + R % G) * D + d]) : 0.f;
  }
}

// Keys (and values) `count` from the page's first on; the places behind them become zero, so that what they hold counts nowhere.
template <typename T>
__device__ __forceinline__ void load_page(Shared& sm, const T* __restrict__ k, const T* __restrict__ v, int count, bool values) {
  constexpr int V = 16 / sizeof(T);  // elements of a 16-byte piece
  if (D % V == 0 && (((uintptr_t)k | (values ? (uintptr_t)v : 0)) & 15) == 0) {
    // a thread's pieces four at a time, so that their loads are on their way together
    constexpr int PIECES = KRK_PAGE * (D / V), AHEAD = 4;
    auto put = [&](float* to, uint4 x) {
      const T* e = reinterpret_cast<const T*>(&x);
#pragma unroll
      for (int c = 0; c < V; c += 4) *reinterpret_cast<float4*>(to + c) = make_float4(to_float<T>(e[c]), to_float<T>(e[c + 1]), to_float<T>(e[c + 2]), to_float<T>(e[c + 3]));
    };
    for (int i0 = threadIdx.x; i0 < PIECES; i0 += THREADS * AHEAD) {
      uint4 kp[AHEAD], vp[AHEAD];
#pragma unroll
      for (int a = 0; a < AHEAD; ++a) {
        const int i = i0 + a * THREADS;
        const bool in = i < PIECES && i / (D / V) < count;
        kp[a] = in ? *reinterpret_cast<const uint4*>(k + (size_t)i * V) : make_uint4(0, 0, 0, 0);
        vp[a] = in && values ? *reinterpret_cast<const uint4*>(v + (size_t)i * V) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int a = 0; a < AHEAD; ++a) {
        const int i = i0 + a * THREADS, key = i / (D / V), d = i % (D / V) * V;
        if (i >= PIECES) break;
        put(&sm.k[key][d], kp[a]);
        if (values) put(&sm.v[key][d], vp[a]);
      }
    }
    return;
  }
  for (int i = threadIdx.x; i < KRK_PAGE * DPAD; i += THREADS) {
    const int key = i / DPAD, d = i % DPAD;
    const bool in = key < count && d < D;
    sm.k[key][d] = in ? to_float<T>(k[key * D + d]) : 0.f;
    if (values) sm.v[key][d] = in ? to_float<T>(v[key * D + d]) : 0.f;
  }
}

// Scores of key threadIdx.x % 64 with eight of the tile's rows, from row 8 * (threadIdx.x / 64) on.
__device__ __forceinline__ void scores(const Shared& sm, float (&s)[8]) {
  const int key = threadIdx.x % KRK_PAGE, r0 = threadIdx.x / KRK_PAGE * 8;
#pragma unroll
  for (int r = 0; r < 8; ++r) s[r] = 0.f;
#pragma unroll 4
  for (int d = 0; d < DPAD; d += 4) {
    const float4 kv = *reinterpret_cast<const float4*>(&sm.k[key][d]);
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const float4 qv = *reinterpret_cast<const float4*>(&sm.q[r0 + r][d]);
      s[r] = fmaf(kv.x, qv.x, fmaf(kv.y, qv.y, fmaf(kv.z, qv.z, fmaf(kv.w, qv.w, s[r]))));
    }
  }
}

// Block (tile x split, kv head, group or sequence): the groups' prefixes first, in n_prefix parts, then the sequences' own keys in
// n_own more.
template <typename T>
__global__ void __launch_bounds__(THREADS)
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
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int last_tok = min(u.n_tok - 1, (tile * TILE + TILE - 1) / G);
  const int key_end = own ? min(u.key_hi, u.start + last_tok + 1) : u.key_hi;  // behind the last key that the tile sees
  int j_lo, j_hi;
  split_pages(u.key_lo, key_end, split, n_splits, j_lo, j_hi);

  load_queries(sm, q, q_stride, u.row0, n_rows, tile, G, kh);
  if (threadIdx.x < TILE) {
    sm.m[threadIdx.x] = -INFINITY;
    sm.l[threadIdx.x] = 0.f;
  }
  float acc[TILE][PER_LANE];
#pragma unroll
  for (int r = 0; r < TILE; ++r)
#pragma unroll
    for (int i = 0; i < PER_LANE; ++i) acc[r][i] = 0.f;

  for (int j = j_lo; j < j_hi; ++j) {
    const int page = seg.table[(size_t)u.slot * seg.width + j];
    const size_t base = ((size_t)page * HKV + kh) * KRK_PAGE * D;
    __syncthreads();  // the page before this one has been read
    load_page(sm, k_cache + base, v_cache + base, min(KRK_PAGE, key_end - j * KRK_PAGE), true);
    __syncthreads();
    {
      float s[8];
      scores(sm, s);
      const int key = threadIdx.x % KRK_PAGE, r0 = threadIdx.x / KRK_PAGE * 8;
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        const int tok = (tile * TILE + r0 + r) / G;
        sm.s[key][r0 + r] = j * KRK_PAGE + key < min(key_end, u.start + tok + 1) ? s[r] * scale_log2 : -INFINITY;
      }
    }
    __syncthreads();
    {
      const int r = threadIdx.x / 8, t = threadIdx.x % 8;  // eight threads a row, neighbours in a warp
      float mx = -INFINITY;
      for (int key = t; key < KRK_PAGE; key += 8) mx = fmaxf(mx, sm.s[key][r]);
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      const float m_old = sm.m[r], m_new = fmaxf(m_old, mx), safe = m_new == -INFINITY ? 0.f : m_new;
      float sum = 0.f;
      const int row_end = min(key_end, u.start + (tile * TILE + r) / G + 1) - j * KRK_PAGE;  // behind the last key of the page that the row sees
      for (int key = t; key < KRK_PAGE; key += 8) {
        const float p = exp2f(sm.s[key][r] - safe);
        sm.s[key][r] = key < row_end ? p : -1.f;  // no weight: what the value is does not count
        if (key < row_end) sum += p;
      }
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      __syncwarp();
      if (t == 0) {
        const float a = exp2f(m_old - safe);
        sm.alpha[r] = a;
        sm.l[r] = sm.l[r] * a + sum;
        sm.m[r] = m_new;
      }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < TILE; ++r) {
      const float a = sm.alpha[r];
#pragma unroll
      for (int i = 0; i < PER_LANE; ++i) acc[r][i] *= a;
    }
    const bool whole = j * KRK_PAGE + KRK_PAGE <= min(key_end, u.start + tile * TILE / G + 1);  // every row sees the page to its end
    for (int key = warp * 16; key < warp * 16 + 16; ++key) {
      float p[TILE];
#pragma unroll
      for (int r = 0; r < TILE; r += 4) *reinterpret_cast<float4*>(p + r) = *reinterpret_cast<const float4*>(&sm.s[key][r]);
#pragma unroll
      for (int i = 0; i < PER_LANE; ++i) {
        const int d = lane + 32 * i;
        const float v = d < DPAD ? sm.v[key][d] : 0.f;
#pragma unroll
        for (int r = 0; r < TILE; ++r)
          if (whole || p[r] >= 0.f || p[r] != p[r]) acc[r][i] = fmaf(p[r], v, acc[r][i]);
      }
    }
  }
  // the four warps' sums, in warp order, through the place of the keys
  __syncthreads();
  float* sum = &sm.k[0][0];  // [TILE][D]
  for (int w = 0; w < THREADS / 32; ++w) {
    if (warp == w) {
#pragma unroll
      for (int r = 0; r < TILE; ++r)
#pragma unroll
        for (int i = 0; i < PER_LANE; ++i) {
          const int d = lane + 32 * i;
          if (d < D) sum[r * D + d] = (w ? sum[r * D + d] : 0.f) + acc[r][i];
        }
    }
    __syncthreads();
  }
  for (int r = 0; r < TILE; ++r) {
    const int R = tile * TILE + r;
    if (R >= n_rows) break;
    const size_t at = parts.at(part0 + split, u.row0 + R / G, kh * G + R % G);
    if (sm.l[r] > 0.f || sm.l[r] != sm.l[r])
      for (int d = threadIdx.x; d < D; d += THREADS) parts.o[at * D + d] = sum[r * D + d];
    if (threadIdx.x == 0) parts.ml[at] = make_float2(sm.m[r], sm.l[r]);
  }
}

// One warp per (row, head): the parts' join. lse (may be null): log2 of the sum of the row's 2^s, for the weights of its keys.
template <typename T>
__global__ void __launch_bounds__(THREADS) join_parts_kernel(T* __restrict__ out, float* __restrict__ lse, Parts parts, int n_parts) {
  grid_launch_dependents();
  grid_dependency_wait();
  const long long item = (long long)blockIdx.x * (THREADS / 32) + (threadIdx.x >> 5);
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
// own. Block (pages x, x + gridDim.x, ..., kv head, sequence); a key's sum is one thread pair's, in the order of the rows.
template <typename T>
__global__ void __launch_bounds__(THREADS)
key_weights_kernel(const float* sums, float* sums_out, int* __restrict__ positions, const int* __restrict__ seq_shift, int capacity,
                   const float* __restrict__ lse, int observe, const T* __restrict__ q, int q_stride, int HQ, int HKV, Segments seg,
                   const T* __restrict__ k_cache, float scale_log2) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  Shared& sm = *reinterpret_cast<Shared*>(smem_raw);
  grid_launch_dependents();
  grid_dependency_wait();
  const int kh = blockIdx.y, seq = blockIdx.z, G = HQ / HKV;
  const Unit u = own_unit(seg, seq);
  const int seen = observe > 0 ? min(observe, u.n_tok) : u.n_tok, tok0 = u.n_tok - seen;
  const int n_rows = seen * G, row0 = u.row0 + tok0;
  const int key = threadIdx.x % KRK_PAGE, half = threadIdx.x / KRK_PAGE;
  for (int j = blockIdx.x; j * KRK_PAGE < u.key_hi; j += gridDim.x) {
    const int page = seg.table[(size_t)u.slot * seg.width + j];
    const size_t base = ((size_t)page * HKV + kh) * KRK_PAGE * D;
    const int at = j * KRK_PAGE + key;
    __syncthreads();
    load_page<T>(sm, k_cache + base, nullptr, min(KRK_PAGE, u.key_hi - j * KRK_PAGE), false);
    float sum = 0.f;
    for (int tile = 0; tile * TILE < n_rows; ++tile) {
      if (u.start + tok0 + min(seen - 1, (tile * TILE + TILE - 1) / G) < j * KRK_PAGE) continue;  // none of its rows sees the page
      __syncthreads();
      load_queries(sm, q, q_stride, row0, n_rows, tile, G, kh);
      if (threadIdx.x < TILE) {
        const int R = tile * TILE + threadIdx.x;
        sm.l[threadIdx.x] = R < n_rows ? lse[(size_t)(row0 + R / G) * HQ + kh * G + R % G] : 0.f;
      }
      __syncthreads();
      float s[8], part = 0.f;
      scores(sm, s);
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        const int R = tile * TILE + half * 8 + r;
        if (R < n_rows && at <= u.start + tok0 + R / G) part += exp2f(fmaf(s[r], scale_log2, -sm.l[half * 8 + r]));
      }
      sum += part;
    }
    __syncthreads();
    if (half == 1) sm.s[key][0] = sum;
    __syncthreads();
    if (half == 0 && at < u.key_hi) {
      sum += sm.s[key][0];
      const size_t place = ((size_t)u.slot * HKV + kh) * capacity + at;
      sums_out[place] = at < u.start ? sums[place] + sum : sum;
      if (positions && at >= u.start) positions[place] = at + (seq_shift ? seq_shift[seq] : 0);
    }
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
  const long long blocks = ((long long)rows * HQ + THREADS / 32 - 1) / (THREADS / 32);
  if (blocks == 0) return 0;
  if (blocks > 0x7fffffffLL) return -3;
  if (dtype == KRK_DTYPE_F32)
    return (int)launch_pdl(join_parts_kernel<float>, dim3((unsigned)blocks), dim3(THREADS), 0, stream, (float*)out, lse, parts, n_parts);
  return (int)launch_pdl(join_parts_kernel<bf16>, dim3((unsigned)blocks), dim3(THREADS), 0, stream, (bf16*)out, lse, parts, n_parts);
}

// page_blocks: blocks that share a sequence's pages; any number is right.
KRK_API int krk_key_weights(const float* sums, float* sums_out, int* positions, const int* seq_shift, int capacity, const float* lse, int observe,
                            const void* q, int q_stride, int HQ, int HKV, KRK_SEGMENTS, const void* k_cache, int page_blocks, float scale, int dtype,
                            cudaStream_t stream) {
  const Segments seg = KRK_MAKE_SEGMENTS;
  if (n_seqs == 0) return 0;
  if (HKV > 65535 || n_seqs > 65535 || page_blocks < 1) return -3;
  const dim3 grid(page_blocks, HKV, n_seqs);
  static unsigned long long allowed[2] = {0, 0};
  auto go = [&](auto* kern, auto* queries, auto* keys) {
    cudaError_t e = allow_shared(kern, SMEM_BYTES, allowed + (dtype == KRK_DTYPE_F32));
    if (e != cudaSuccess) return (int)e;
    return (int)launch_pdl(kern, grid, dim3(THREADS), SMEM_BYTES, stream, sums, sums_out, positions, seq_shift, capacity, lse, observe, queries,
                           q_stride, HQ, HKV, seg, keys, scale * LOG2E);
  };
  if (dtype == KRK_DTYPE_F32) return go(key_weights_kernel<float>, (const float*)q, (const float*)k_cache);
  return go(key_weights_kernel<bf16>, (const bf16*)q, (const bf16*)k_cache);
}

// Attention in parts and their join (out; lse may be null) and, where sums_out is given, the weights of the keys, with lse as their logarithms: krk_partial_attention,
// krk_join_parts and krk_key_weights in one call. o, ml: scratch for n_prefix + n_own parts.
KRK_API int krk_attention_in_parts(void* out, float* lse, float* o, float* ml, int rows, int n_prefix, int n_own, const float* sums, float* sums_out,
                                   int* positions, const int* seq_shift, int capacity, int observe, int page_blocks, const void* q, int q_stride, int HQ,
                                   int HKV, KRK_SEGMENTS, const void* k_cache, const void* v_cache, int group_rows, int own_rows, float scale, int dtype,
                                   cudaStream_t stream) {
  int rc = krk_partial_attention(o, ml, rows, n_prefix, n_own, q, q_stride, HQ, HKV, cu_q, seq_slot, seq_start, seq_qlen, group_cu, group_len, seq_group,
                                 n_seqs, n_groups, table, width, k_cache, v_cache, group_rows, own_rows, scale, dtype, stream);
  if (rc == 0) rc = krk_join_parts(out, lse, o, ml, rows, HQ, n_prefix + n_own, dtype, stream);
  if (rc == 0 && sums_out)
    rc = krk_key_weights(sums, sums_out, positions, seq_shift, capacity, lse, observe, q, q_stride, HQ, HKV, cu_q, seq_slot, seq_start, seq_qlen, group_cu,
                         group_len, seq_group, n_seqs, n_groups, table, width, k_cache, page_blocks, scale, dtype, stream);
  return rc;
}
