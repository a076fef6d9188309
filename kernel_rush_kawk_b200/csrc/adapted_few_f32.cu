// The float32 product of up to 16 rows (few_f32.cuh) with the rows' low-rank adapters: t is made by a launch that the weights' copies begin beside, and a thread
// adds the second factor to the sum that it holds. The result has the bits of the three launches that more rows take (adapters.cu).
// Bound as the product alone is, which takes twice its bytes' time there (its chains of 2,560 multiply-adds at four clocks are 5 us of it): six rows of 2,560 x 6,144, four adapters of rank 8, cold and replayed 22.5 to 24.5
// us (the product alone 22.5; 64 MB, 9.8 us), a call 18.6 where three launches took 28.7.
#include <climits>

#include "adapters.cuh"
#include "few_f32.cuh"

namespace {

struct AdapterMore {
  static constexpr bool ON = true;
  AdapterBank bank;
  const float* t;
  const int* row_adapter;

  // B's rows into L2 while the weights stream (row_adapter is an earlier kernel's than the first factor's, which was waited for before this one began)
  __device__ void ask(int r, int n) const {
    const int a = row_adapter[r];
    if (a < 0 || a >= bank.capacity) return;
    const float* b = reinterpret_cast<const float*>(bank.b) + ((size_t)a * bank.begin[KRK_MAX_PARTS] + n) * bank.rank;
    for (int j = 0; j < bank.rank; j += 32) asm volatile("prefetch.global.L2 [%0];" ::"l"(b + j));
  }
  __device__ void wait() const {
    grid_dependency_wait();
    grid_launch_dependents();
  }
  // the sums of R rows from row0 and the C columns n
  template <int R, int C> __device__ void add(float (&sums)[R][C], int row0, int rows, const int (&n)[C]) const {
    int a[R], row[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      row[r] = min(row0 + r, rows - 1);
      a[r] = row0 + r < rows ? row_adapter[row[r]] : -1;
      if (a[r] >= bank.capacity) a[r] = -1;
    }
    add_second_factor<float, R, C>(bank, t, a, row, n, sums);
  }
};

}  // namespace

// out [rows, N] float32 from x [rows, K] (row stride ldx) and w [N, K] (row stride ldw), up to 16 rows. K and the strides are multiples of 4. t: float32 scratch of
// rows * parts * wide.
KRK_API int krk_adapted_few_f32(float* out, const float* x, long long ldx, const float* w, long long ldw, int rows, int N, int K, const AdapterBank* bank, const int* row_adapter,
                                float* t, int* error, cudaStream_t stream) {
  if (rows == 0 || N == 0) return 0;
  if (rows > 16 || ldx > INT_MAX || ldw > INT_MAX || K < 4 || K % 4 || ldx % 4 || ldw % 4 || bank->begin[KRK_MAX_PARTS] != N ||
      (((uintptr_t)x | (uintptr_t)w | (uintptr_t)out | (uintptr_t)bank->b | (uintptr_t)t) & 15))
    return -2;
  const int rc = krk_first_factor_f32(t, x, ldx, rows, K, *bank, row_adapter, error, KRK_DTYPE_F32, stream);
  return rc ? rc : launch_f32_few(out, x, w, rows, N, K, (int)ldx, (int)ldw, N, error, AdapterMore{*bank, t, row_adapter}, stream);
}
