// What the kernels of the low-rank adapters share: how a bank of adapters lies in memory, and which rows of a step are whose.
//
// A projection of N outputs over K inputs has `parts` (queries, keys and values beside one another, say; at most four), part p the outputs
// begin[p] <= n < begin[p + 1]. A bank holds for adapter `a` the first factors A [parts * rank, K], the second factors B [N, rank] and for
// each part the rank in use (0: the adapter leaves the part as it is) and the scale:
//   y[r, n] = sum_k x[r, k] W[n, k] + scale[a, p] sum_j B[a, n, j] (sum_k x[r, k] A[a, p * rank + j, k])      a = row_adapter[r], p of n
// Rows whose adapter is negative have none. An adapter that the bank does not hold sets the error word and counts as none.
#pragma once

#include "common.cuh"

#define KRK_MAX_PARTS 4
#define KRK_ERROR_ADAPTER 26  // a row's adapter is none of the bank's
#define KRK_ERROR_MAPS 27     // lengths, slots or pages that do not fit the step

struct AdapterBank {
  const void* a;       // [capacity, parts * rank, K]
  const void* b;       // [capacity, N, rank]
  const float* scale;  // [capacity, parts]
  const int* ranks;    // [capacity, parts]
  int capacity, parts, rank;
  int begin[KRK_MAX_PARTS + 1];
  int wide;            // columns of t for a part: rank, up to the next multiple of 16
};

// The rows in tiles, and the adapters that a tile's rows have: tile i has info[2 * i + 1] of them, in the slots from info[2 * i] on. A slot has an adapter
// and its tile; -1 for a slot that is not used.
struct AdapterTiles {
  const int* row_adapter;  // [rows]
  const int* info;         // [tiles, 2]
  const int* slots;        // [n_slots, 2]
  int rows, tile_rows, n_slots;
};

__device__ __forceinline__ int part_of(const AdapterBank& bank, int n) {
  int p = 0;
#pragma unroll
  for (int i = 1; i < KRK_MAX_PARTS; ++i) p += (i < bank.parts && n >= bank.begin[i]);
  return p;
}

// sums[r][c] += sum_j t[r, p of n, j] B[a, n, j] in 32 bits for R rows and C columns at once (a[r] negative: nothing; n[c] negative: not there), the factors' sum one
// chain over j, added to what is there at the end; t float32 [rows, parts * wide]. Sixteen j of all of them are read before they are multiplied: one output
// after another took 13 us behind sixteen rows of rank 64.
template <typename T, int R, int C>
__device__ __forceinline__ void add_second_factor(const AdapterBank& bank, const float* t, const int (&a)[R], const int (&row)[R], const int (&n)[C], float (&sums)[R][C]) {
  const T* b[R][C];
  const float* tr[R][C];
  int rank[R][C], most = 0;
  float sum[R][C];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const bool there = a[r] >= 0 && n[c] >= 0;
      const int p = there ? part_of(bank, n[c]) : 0;
      rank[r][c] = there ? bank.ranks[a[r] * bank.parts + p] : 0;
      b[r][c] = reinterpret_cast<const T*>(bank.b) + ((size_t)max(a[r], 0) * bank.begin[KRK_MAX_PARTS] + max(n[c], 0)) * bank.rank;
      tr[r][c] = t + ((size_t)row[r] * bank.parts + p) * bank.wide;
      most = max(most, rank[r][c]);
      sum[r][c] = 0.f;
    }
  constexpr int AT_ONCE = R * C > 2 ? 8 : 16;
#pragma unroll 1
  for (int j = 0; j < most; j += AT_ONCE) {
    __align__(16) float u[R][C][AT_ONCE], v[R][C][AT_ONCE];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < AT_ONCE; i += 4) {
          const bool in = j + i < rank[r][c];  // (the bank's rank is a multiple of eight, and both factors are zeros behind the adapter's)
          *reinterpret_cast<float4*>(&u[r][c][i]) = in ? __ldcg(reinterpret_cast<const float4*>(tr[r][c] + j + i)) : make_float4(0.f, 0.f, 0.f, 0.f);
          if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<float4*>(&v[r][c][i]) = in ? *reinterpret_cast<const float4*>(b[r][c] + j + i) : make_float4(0.f, 0.f, 0.f, 0.f);
          } else {
            const uint2 two = in ? *reinterpret_cast<const uint2*>(b[r][c] + j + i) : make_uint2(0, 0);
            v[r][c][i] = __uint_as_float(two.x << 16);
            v[r][c][i + 1] = __uint_as_float(two.x & 0xffff0000u);
            v[r][c][i + 2] = __uint_as_float(two.y << 16);
            v[r][c][i + 3] = __uint_as_float(two.y & 0xffff0000u);
          }
        }
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i)
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int c = 0; c < C; ++c) sum[r][c] = fmaf(u[r][c][i], v[r][c][i], sum[r][c]);
  }
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (rank[r][c] > 0) sums[r][c] += sum[r][c];
}

// t = scale (x A^T) of every slot, or (compact) of every row that has an adapter (first_factor.cu); sets n_done words at `done` to zero. Lets the next kernel start
// once what came before is over: that one may read what earlier kernels wrote before it waits, and waits before it reads t.
int krk_first_factor(void* t, bool compact, int* done, int n_done, const void* x, long long ldx, int K, const AdapterBank& bank, const AdapterTiles& tiles, int* error,
                     cudaStream_t stream);
// The same in 32 bits, for every type: t [rows, parts * wide] float32 of every row that has an adapter (adapters.cu). Lets the next kernel start as above.
int krk_first_factor_f32(float* t, const void* x, long long ldx, int rows, int K, const AdapterBank& bank, const int* row_adapter, int* error, int dtype,
                         cudaStream_t stream);
