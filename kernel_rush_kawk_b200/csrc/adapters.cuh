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

// t = scale (x A^T) of every slot, or (compact) of every row that has an adapter (first_factor.cu); sets n_done words at `done` to zero. Lets the next kernel start
// once what came before is over: that one may read what earlier kernels wrote before it waits, and waits before it reads t.
int krk_first_factor(void* t, bool compact, int* done, int n_done, const void* x, long long ldx, int K, const AdapterBank& bank, const AdapterTiles& tiles, int* error,
                     cudaStream_t stream);
