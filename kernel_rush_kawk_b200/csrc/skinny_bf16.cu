// The decode-time product for few rows (skinny.cuh) as this library's entry.
#define KRK_TRACE_OWNER  // with -DKRK_TRACE this file keeps the timeline buffer
#include "skinny.cuh"

#ifdef KRK_TRACE
KRK_API int krk_trace_dump(unsigned long long* host, unsigned int cap, unsigned int* count) {
  cudaDeviceSynchronize();
  cudaMemcpyFromSymbol(count, krk_trace_count, sizeof(unsigned int));
  unsigned int n = *count < cap ? *count : cap;
  if (n > KRK_TRACE_CAP) n = KRK_TRACE_CAP;
  cudaMemcpyFromSymbol(host, krk_trace_buf, (size_t)n * 4 * sizeof(unsigned long long));
  unsigned int zero = 0;
  cudaMemcpyToSymbol(krk_trace_count, &zero, sizeof(unsigned int));
  return 0;
}
#endif

// out [M, N] (bfloat16 or float32), x [M, K] bfloat16 contiguous, W [N, K] ([2N, K] with a gate) bfloat16
// contiguous. Needs M <= 16 and K % 32 == 0. gate: 0 none, 1 SwiGLU, 2 the tanh form of GELU, 3 gate and up clamped
// at `limit`, swish with slope 1.702 times (up + 1), 4 no gate but the squared relu of the plain product.
KRK_API int krk_skinny_linear(void* out, const void* x, const void* W, int M, int N, int K, float limit, int gate,
                              int out_dtype, cudaStream_t stream) {
  if (M == 0 || N == 0) return 0;
  if (M > 16 || K % CHUNK || K <= 0) return -2;
  if (gate != 0 && out_dtype != KRK_DTYPE_BF16) return -4;
  if (gate == 4) return pick_nt<0, bf16>(out, x, W, M, N, K, -1.f, stream);
  if (gate == 3) return pick_nt<3, bf16>(out, x, W, M, N, K, limit, stream);
  if (gate == 2) return pick_nt<2, bf16>(out, x, W, M, N, K, 0.f, stream);
  if (gate) return pick_nt<1, bf16>(out, x, W, M, N, K, 0.f, stream);
  if (out_dtype == KRK_DTYPE_F32) return pick_nt<0, float>(out, x, W, M, N, K, 0.f, stream);
  return pick_nt<0, bf16>(out, x, W, M, N, K, 0.f, stream);
}
