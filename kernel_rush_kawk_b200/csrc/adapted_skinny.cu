// The product of few rows (skinny.cuh) with the rows' low-rank adapters: the weights stream while the first factor's kernel (first_factor.cu) makes t, and every adapter
// that the rows have is a few more steps of k behind them, B's rows in the weights' place and t, zero for rows that have another adapter, in the rows'. Up to 16
// rows are the weights' bytes and little else; what the adapters add is a launch that the weights' loads run beside, and the wait for t and for
// B, which is asked into L2 at a block's beginning. t is rounded to bfloat16 (half a step of 2^-8 of a sum that is itself a part of the result, which
// is rounded the same way), nothing else on the way to the result.
//
// Bound by memory. Cold and replayed, less what an empty replay takes (4.1 us): one row of 2,560 x 6,144 8 to 9 us, as the product alone (31 MB, 4.8), eight rows with
// five adapters of rank 16 of 4,096 x 2,560 10.2 (alone 6 to 8), 16 rows with nine, gate and up of 2,560 x 19,456 24.6 (alone 22.5; 102 MB, 16). In a step that is
// replayed, where the product alone loads its weights beside the kernel before it, the first factor's launch stands between: 4.3 us a product at one row.
// (Letting the weights' loads in before the first factor has waited, and waiting for it before x is read, made that 6.9; having W's first 16 MB asked into L2 by
// the first factor's waiting blocks 17.) Five blocks of four warps share an SM, so 96 registers: in 102, of 608 blocks 16 ran behind the others, 41 us for 34.8.
#include "adapters.cuh"
#include "skinny.cuh"

namespace {

struct AdapterSteps {
  static constexpr bool ON = true;
  struct Row {
    int count, listed;  // adapters of the rows; the lane's one
    int mine[2];        // the adapters of the rows that this lane has in the batch's fragments
  };
  AdapterBank bank;
  const bf16* t;  // [M, parts * wide]
  AdapterTiles tiles;
  int* error;

  // the tiles' first rows of W, and the rows that there are
  template <int RT> __device__ static int tile_row(int s, int N, int n0, bool gated, int& end) {
    end = gated && s >= RT ? 2 * N : N;
    return n0 + s % RT * 16 + (gated && s >= RT ? N : 0);
  }

  template <int TILES, int NT, int RT> __device__ Row begin(int M, int N, int n0, bool gated, int id, int ids) const {
    const int lane = threadIdx.x & 31;
    Row row;
    row.count = tiles.info[1];
    row.listed = lane < 16 ? tiles.slots[2 * min(lane, tiles.n_slots - 1)] : -1;
#pragma unroll
    for (int j = 0; j < NT; ++j) row.mine[j] = 8 * j + (lane >> 2) < M ? tiles.row_adapter[8 * j + (lane >> 2)] : -1;
    if (lane >= row.count) row.listed = -1;
    if (row.listed >= bank.capacity) {
      atomicExch(error, KRK_ERROR_ADAPTER);
      row.listed = -1;
    }
    for (int i = id; i < row.count; i += ids) {
      const int a = __shfl_sync(0xffffffffu, row.listed, i);
      if (a < 0) continue;
#pragma unroll
      for (int s = 0; s < TILES; ++s) {
        int end;
        const int n = tile_row<RT>(s, N, n0, gated, end) + lane % 16;
        if (lane < 16 && n < end)
          asm volatile("prefetch.global.L2 [%0];" ::"l"(reinterpret_cast<const bf16*>(bank.b) + ((size_t)a * bank.begin[KRK_MAX_PARTS] + n) * bank.rank));
      }
    }
    return row;
  }

  template <int TILES, int NT, int RT> __device__ void add(const Row& row, float (&acc)[TILES][NT][4], int N, int n0, bool gated, int id, int ids) const {
    const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
    const uint4 zero = make_uint4(0, 0, 0, 0);
    for (int i = id; i < row.count; i += ids) {
      const int a = __shfl_sync(0xffffffffu, row.listed, i);
      if (a < 0) continue;
#pragma unroll
      for (int s = 0; s < TILES; ++s) {
        int end;
        const int n = tile_row<RT>(s, N, n0, gated, end);
        if (n >= end) continue;
        const int last = part_of(bank, min(n + 16, end) - 1);
        for (int p = part_of(bank, n); p <= last; ++p) {  // (one, but where a tile reaches over a border)
          const int rank = bank.ranks[a * bank.parts + p];
          const bool row0 = n + g >= bank.begin[p] && n + g < min(end, bank.begin[p + 1]), row1 = n + g + 8 >= bank.begin[p] && n + g + 8 < min(end, bank.begin[p + 1]);
          const bf16* b = reinterpret_cast<const bf16*>(bank.b) + ((size_t)a * bank.begin[KRK_MAX_PARTS] + n + g) * bank.rank + 8 * q;
          for (int k = 0; k < rank; k += 32) {  // (behind the rank, up to the bank's, both factors are zeros)
            const bool in = k + 8 * q < bank.rank;
            const uint4 w0 = in && row0 ? ld_stream_16(b + k) : zero, w1 = in && row1 ? ld_stream_16(b + (size_t)8 * bank.rank + k) : zero;
#pragma unroll
            for (int j = 0; j < NT; ++j) {
              const uint4 x = in && row.mine[j] == a ? __ldcg(reinterpret_cast<const uint4*>(t + ((size_t)(8 * j + g) * bank.parts + p) * bank.wide + k + 8 * q)) : zero;
              mma_bf16_16816(acc[s][j], w0.x, w1.x, w0.y, w1.y, x.x, x.y);
              mma_bf16_16816(acc[s][j], w0.z, w1.z, w0.w, w1.w, x.z, x.w);
            }
          }
        }
      }
    }
  }
};

}  // namespace

// out [rows, N] (gated: [rows, N / 2]) bfloat16 from x [rows, K] and w [N, K], both contiguous, up to 16 rows in one tile. K is a multiple of 32. t: bfloat16 scratch
// of rows * parts * wide.
KRK_API int krk_adapted_skinny(void* out, const void* x, const void* w, int rows, int N, int K, const AdapterBank* bank, const int* row_adapter, const int* info,
                               const int* slots, int n_slots, int tile_rows, void* t, int gated, int* error, cudaStream_t stream) {
  if (rows == 0 || N == 0) return 0;
  if (rows > 16 || rows > tile_rows || K % 32 || K < 64 || n_slots < 1 || bank->begin[KRK_MAX_PARTS] != N ||
      (((uintptr_t)x | (uintptr_t)w | (uintptr_t)bank->a | (uintptr_t)bank->b | (uintptr_t)t) & 15))
    return -2;
  const AdapterTiles tiles = {row_adapter, info, slots, rows, tile_rows, n_slots};
  const int rc = krk_first_factor(t, true, nullptr, 0, x, K, K, *bank, tiles, error, stream);
  if (rc) return rc;
  const AdapterSteps steps = {*bank, (const bf16*)t, tiles, error};
  return gated ? pick_nt<1, bf16>(out, x, w, rows, N / 2, K, 0.f, stream, steps) : pick_nt<0, bf16>(out, x, w, rows, N, K, 0.f, stream, steps);
}
