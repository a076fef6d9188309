// Attention in parts for steps of many tokens, bfloat16, on the warp-level tensor cores (partial_attention.cuh says what the parts are):
// a sequence's new tokens over its own keys, causally, joined with the parts of the prefix that they share; and, where asked
// for, the logarithm of every row's sum, by which the weights of its keys can be had again.
//
// A block takes 64 (token, head) rows of one kv head, 16 a warp, and walks the pages that the tile sees, two in shared memory (cp.async).
// The keys behind a shared prefix are few beside it, which is where the time goes (prefix_tcgen05.cu): this kernel's share of
// sixteen questions of up to 90 tokens behind 4,096 positions is a sixth, 16 of 92 us, most of it the join's reading of the parts (47 MB).
//
// Values that a row does not see may be anything, and zero times infinity is not zero: values behind the sequence's end count
// as zero, and a page that some row sees in part and that holds an infinity or a NaN goes through the multiplications one by one.
//
// P is rounded to bfloat16 before it meets the values, as everywhere on this path; scores, statistics and sums are float32.
//
// Compiled once per head size: -DKRK_HEAD_DIM=<D>.
#include "mma.cuh"
#include "partial_attention.cuh"

#ifndef KRK_HEAD_DIM
#error "compile with -DKRK_HEAD_DIM=<head size>"
#endif

#if KRK_HEAD_DIM % 16 == 0 && KRK_HEAD_DIM <= 256

namespace {

#include "attention_tiles.cuh"

// The weights of a page with values that are no numbers, [64 rows][64 keys], lie where its keys were, or behind the pages where keys are too small.
constexpr bool WEIGHTS_IN_KEYS = TILE_ELEMS >= 64 * KRK_PAGE;
constexpr size_t WEIGHTS_BYTES = WEIGHTS_IN_KEYS ? 0 : (size_t)64 * KRK_PAGE * sizeof(bf16);

__device__ __forceinline__ bool not_finite(uint32_t two) { return (two & 0x7f80u) == 0x7f80u || (two & 0x7f800000u) == 0x7f800000u; }

__global__ void __launch_bounds__(THREADS, D <= 128 ? 3 : 1)
many_rows_kernel(bf16* __restrict__ out, float* __restrict__ lse, Parts parts, int n_join, const bf16* __restrict__ q, int q_stride, int HQ, int HKV,
                 Segments seg, const bf16* __restrict__ k_cache, const bf16* __restrict__ v_cache, float scale_log2, bool wait_first) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  bf16* smem = reinterpret_cast<bf16*>(smem_raw);                          // [2 stages][K, V][64][pitch]
  if (wait_first) grid_dependency_wait();
  grid_launch_dependents();
  const int kh = blockIdx.y, G = HQ / HKV;
  const int tile = gridDim.x - 1 - blockIdx.x;  // long tiles first
  const Unit u = own_unit(seg, blockIdx.z);
  const int n_rows = u.n_tok * G;
  if (tile * 64 >= n_rows) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t4 = lane & 3;

  int tok[2], pos[2];
  const bf16* qp[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int R = tile * 64 + warp * 16 + g + 8 * h;
    const bool ok = R < n_rows;
    tok[h] = ok ? R / G : -1;
    pos[h] = ok ? u.start + tok[h] : -1;  // -1: sees nothing
    qp[h] = ok ? q + (size_t)(u.row0 + tok[h]) * q_stride + (size_t)(kh * G + R % G) * D : nullptr;
  }
  uint32_t qf[KSTEPS][4];
  load_q(qf, qp[0], qp[1], lane);
  int warp_min_pos = min(pos[0], pos[1]);
#pragma unroll
  for (int o2 = 16; o2 > 0; o2 >>= 1) warp_min_pos = min(warp_min_pos, __shfl_xor_sync(0xffffffffu, warp_min_pos, o2));
  const int tile_min_pos = u.start + tile * 64 / G;  // the least position of the tile's rows

  const int last_tok = min(u.n_tok - 1, (tile * 64 + 63) / G);
  const int j_lo = u.key_lo / KRK_PAGE, j_hi = min(u.start + last_tok, u.key_hi - 1) / KRK_PAGE;
  const size_t page_stride = (size_t)HKV * KRK_PAGE * D, head_off = (size_t)kh * KRK_PAGE * D;
  auto issue = [&](int j, int stage) {
    const int page = seg.table[(size_t)u.slot * seg.width + j];
    bf16* ks = smem + (size_t)stage * 2 * TILE_ELEMS;
    load_page(ks, k_cache + (size_t)page * page_stride + head_off);
    load_page(ks + TILE_ELEMS, v_cache + (size_t)page * page_stride + head_off);
    cp_async_commit();
  };

  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  float o[DTILES][4];
#pragma unroll
  for (int n = 0; n < DTILES; ++n)
#pragma unroll
    for (int c = 0; c < 4; ++c) o[n][c] = 0.f;

  if (j_lo <= j_hi) issue(j_lo, 0);
  for (int j = j_lo; j <= j_hi; ++j) {
    const int stage = (j - j_lo) & 1, key_base = j * KRK_PAGE;
    if (j + 1 <= j_hi) {
      issue(j + 1, stage ^ 1);
      cp_async_wait<1>();
    } else {
      cp_async_wait<0>();
    }
    __syncthreads();
    bf16* ks = smem + (size_t)stage * 2 * TILE_ELEMS;
    bf16* vs = ks + TILE_ELEMS;
    bool one_by_one = false;
    if (key_base + KRK_PAGE - 1 > tile_min_pos) {  // some row sees the page in part: what do the values hold that it does not see?
      const int count = u.key_hi - key_base;       // of the sequence's
      bool odd = false;
      for (int e = threadIdx.x; e < KRK_PAGE * (D / 8); e += THREADS) {
        uint4* at = reinterpret_cast<uint4*>(vs + kv_off(e / (D / 8), e % (D / 8)));
        if (e / (D / 8) >= count) {
          *at = make_uint4(0, 0, 0, 0);
        } else {
          const uint4 x = *at;
          odd |= not_finite(x.x) || not_finite(x.y) || not_finite(x.z) || not_finite(x.w);
        }
      }
      one_by_one = __syncthreads_or(odd);
    }
    float s[8][4];
    qk_tile<8>(s, qf, ks, 0, lane);
    const bool whole = key_base + KRK_PAGE - 1 <= warp_min_pos;
#pragma unroll
    for (int n = 0; n < 8; ++n)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const bool seen = whole || key_base + n * 8 + 2 * t4 + (c & 1) <= pos[c >> 1];
        s[n][c] = seen ? s[n][c] * scale_log2 : -INFINITY;
      }
    softmax_update<8>(s, m, l, o);
    if (!one_by_one) {
      pv_tile<8>(o, s, vs, 0, lane);
    } else {
      bf16* weights = WEIGHTS_IN_KEYS ? ks : reinterpret_cast<bf16*>(smem_raw + PAGE_SMEM);
      __syncthreads();  // every warp has its scores
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int n = 0; n < 8; ++n)
          *reinterpret_cast<uint32_t*>(weights + (warp * 16 + g + 8 * h) * KRK_PAGE + n * 8 + 2 * t4) = pack_bf16x2(s[n][2 * h], s[n][2 * h + 1]);
      __syncwarp();
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const bf16* row = weights + (warp * 16 + g + 8 * h) * KRK_PAGE;
        for (int key = 0; key < KRK_PAGE && key_base + key <= pos[h]; ++key) {
          const float p = __bfloat162float(row[key]);
#pragma unroll
          for (int n = 0; n < DTILES; ++n) {
            const bf16* v = vs + kv_off(key, n) + 2 * t4;
            o[n][2 * h] = fmaf(p, __bfloat162float(v[0]), o[n][2 * h]);
            o[n][2 * h + 1] = fmaf(p, __bfloat162float(v[1]), o[n][2 * h + 1]);
          }
        }
      }
    }
    __syncthreads();  // the stage is free for the load after next
  }

  if (!wait_first) grid_dependency_wait();  // the prefix parts are there
  const size_t part_step = (size_t)parts.rows * parts.HQ;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (tok[h] < 0) continue;
    const int head = kh * G + (tile * 64 + warp * 16 + g + 8 * h) % G;
    const size_t item = (size_t)(u.row0 + tok[h]) * HQ + head;
    float big = m[h], total = l[h];
    for (int p = 0; p < n_join; ++p) big = fmaxf(big, parts.ml[p * part_step + item].x);
    const float safe = big == -INFINITY ? 0.f : big;
    if (n_join > 0) {
      const float w = exp2f(m[h] - safe);
      total *= w;
#pragma unroll
      for (int n = 0; n < DTILES; ++n) { o[n][2 * h] *= w; o[n][2 * h + 1] *= w; }
    }
    for (int p = 0; p < n_join; ++p) {
      const float2 ml = parts.ml[p * part_step + item];
      if (ml.y == 0.f) continue;
      const float w = exp2f(ml.x - safe);
      total += w * ml.y;
#pragma unroll
      for (int n = 0; n < DTILES; ++n) {
        const float2 v = *reinterpret_cast<const float2*>(parts.o + (p * part_step + item) * D + n * 8 + 2 * t4);
        o[n][2 * h] += w * v.x;
        o[n][2 * h + 1] += w * v.y;
      }
    }
    const float inv = 1.f / total;
#pragma unroll
    for (int n = 0; n < DTILES; ++n)
      *reinterpret_cast<uint32_t*>(out + item * D + n * 8 + 2 * t4) = pack_bf16x2(o[n][2 * h] * inv, o[n][2 * h + 1] * inv);
    if (lse && t4 == 0) lse[item] = safe + log2f(total);
  }
}

}  // namespace

// Any number of tokens a sequence: its own keys (all, without groups), joined with the prefix parts 0 .. n_join - 1, which the launch before
// this one writes (n_join 0: none, and the launch before may write the rows and keys themselves). lse: [rows][HQ] or null.
KRK_API int krk_own_rows(void* out, float* lse, const float* o, const float* ml, int rows, int n_join, const void* q, int q_stride, int HQ, int HKV,
                         const int* cu_q, const int* seq_slot, const int* seq_start, const int* seq_qlen, const int* group_cu, const int* group_len,
                         const int* seq_group, int n_seqs, int n_groups, const int* table, int width, const void* k_cache, const void* v_cache,
                         int max_q_len, float scale, cudaStream_t stream) {
  if (rows == 0 || n_seqs == 0 || max_q_len == 0) return 0;
  const long long tiles = ((long long)max_q_len * (HQ / HKV) + 63) / 64;
  if (tiles > 0x7fffffffLL || HKV > 65535 || n_seqs > 65535) return -3;
  const size_t smem = PAGE_SMEM + WEIGHTS_BYTES;
  static unsigned long long allowed = 0;
  cudaError_t e = allow_shared(many_rows_kernel, smem, &allowed);
  if (e != cudaSuccess) return (int)e;
  const Parts parts = {const_cast<float*>(o), (float2*)const_cast<float*>(ml), rows, HQ};
  const Segments seg = {cu_q, seq_slot, seq_start, seq_qlen, group_cu, group_len, seq_group, n_seqs, n_groups, table, width};
  return (int)launch_pdl(many_rows_kernel, dim3((unsigned)tiles, HKV, n_seqs), dim3(THREADS), smem, stream, (bf16*)out, lse, parts, n_join,
                         (const bf16*)q, q_stride, HQ, HKV, seg, (const bf16*)k_cache, (const bf16*)v_cache, scale * LOG2E, n_join == 0);
}

#endif  // head sizes served by this kernel
