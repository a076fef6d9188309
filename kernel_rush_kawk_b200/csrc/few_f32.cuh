// Up to 16 float32 rows times a matrix of float32 weights, every sum one chain of multiply-adds over k, on the CUDA cores.
//
// Bound by the weights' bytes: each is read once, by bulk copies a slice or two ahead; a thread owns one or two output columns of one or two
// rows. One row of 151,936 x 2,560: 235 us, 6.6 TB/s; three rows 226, of 2,560 x 9,728 35 us, where the chain of K multiply-adds is the bound
// (20 us at four clocks each; copies of 16 bytes by all threads: 265 and 46; the general kernel: 1.9 ms and 570 us of 2,560 x 4,096).
//
// `More` is what a program puts behind the sums (nothing: NoMore): ask() at a block's beginning, wait() and add() at its end.
#pragma once

#include "mma.cuh"      // the cache policy of streamed weights
#include "tcgen05.cuh"  // mbarriers

namespace {

// ---- float32, up to 16 rows ------------------------------------------------------------------------------------
// A block owns 16 * CPT columns (a thread c, c + 16); a group of 16 threads takes RPT rows, a warp has two groups, and there are as many
// warps as the rows ask for. A slice is SLICE k of the columns' weights and of the rows. One more warp asks for slices, a bulk copy a
// column (1 KB), as far ahead as the ring is deep, so that the others only wait and multiply: with 16-byte copies by all threads, asking
// for a slice took 600 to 1,200 clocks of the 1,200 that its 256 multiply-adds take in their chain (256 x 4, and the reads).
// Beyond 8 rows, where shared-memory reads are the bound, a thread's two rows of two columns read half as much for a
// multiply-add as one of one.
constexpr int FEW_MAX_DEPTH = 3;
constexpr int FEW_BARS = 2 * FEW_MAX_DEPTH * 8;  // bytes before the ring: slice is here, slice is free

struct NoMore {
  static constexpr bool ON = false;
};

template <int RPT, int CPT, int SLICE, typename More>
__global__ void __launch_bounds__(160)
gemm_f32_few_kernel(float* __restrict__ C, const float* __restrict__ A, const float* __restrict__ W, int M, int N, int K,
                    int lda, int ldw, int ldc, int depth, int* __restrict__ error, const __grid_constant__ More more) {
  constexpr int COLS = 16 * CPT, PITCH = SLICE + 4;
  extern __shared__ __align__(16) unsigned char smem[];
  uint64_t* full = reinterpret_cast<uint64_t*>(smem);
  uint64_t* free_ = full + FEW_MAX_DEPTH;
  float* ring = reinterpret_cast<float*>(smem + FEW_BARS);
  const int stage_floats = (COLS + M) * PITCH;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, readers = (blockDim.x >> 5) - 1;
  const int n0 = blockIdx.x * COLS;
  const int slices = (K + SLICE - 1) / SLICE;
  if (tid == 0) {
    for (int i = 0; i < depth; ++i) {
      tc::mbar_init(full + i, 1);
      tc::mbar_init(free_ + i, readers);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  if (warp == readers) {  // the copies: a lane has columns (or rows) lane, lane + 32 of a slice
    const int cols = min(COLS, N - n0);
    const uint64_t policy = l2_evict_first_policy();
    for (int s = 0, b = 0, round = 0; s < slices; ++s) {
      if (round > 0 && !__all_sync(0xffffffffu, tc::mbar_wait(free_ + b, (round - 1) & 1))) {  // a reader has given up, and says so
        tc::wait_for_copies(full, depth, s);
        return;
      }
      const int bytes = min(SLICE, K - s * SLICE) * 4;
      if (lane == 0) tc::mbar_expect_tx(full + b, (cols + M) * bytes);
      __syncwarp();
      float* dst = ring + b * stage_floats;
      for (int r = lane; r < cols; r += 32)
        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;"
                     ::"r"(tc::smem_u32(dst + r * PITCH)), "l"(W + (size_t)(n0 + r) * ldw + s * SLICE), "r"(bytes), "r"(tc::smem_u32(full + b)), "l"(policy)
                     : "memory");
      if (lane < M)
        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                     ::"r"(tc::smem_u32(dst + (COLS + lane) * PITCH)), "l"(A + (size_t)lane * lda + s * SLICE), "r"(bytes), "r"(tc::smem_u32(full + b))
                     : "memory");
      if (++b == depth) { b = 0; ++round; }
    }
    return;  // what has been asked for is read, or waited for by the reader that gives up
  }
  // neighbouring lanes share a column and differ in their rows
  const int col = lane >> 1, group = 2 * warp + (lane & 1);
  float acc[RPT][CPT];
#pragma unroll
  for (int r = 0; r < RPT; ++r)
#pragma unroll
    for (int c = 0; c < CPT; ++c) acc[r][c] = 0.f;
  const int row0 = group * RPT;
  if constexpr (More::ON)
#pragma unroll
    for (int r = 0; r < RPT; ++r)
#pragma unroll
      for (int c = 0; c < CPT; ++c)
        if (row0 + r < M && n0 + col + 16 * c < N) more.ask(row0 + r, n0 + col + 16 * c);
  int xat[RPT];
#pragma unroll
  for (int r = 0; r < RPT; ++r) xat[r] = (COLS + min(row0 + r, M - 1)) * PITCH;
  bool here = true;
  for (int s = 0, b = 0, round = 0; s < slices; ++s) {
    // a wait that runs out: the warp's outputs are NaN
    here = __all_sync(0xffffffffu, tc::mbar_wait(full + b, round & 1));
    if (!here) {  // a place that it hands back no more is not filled again: what may be on its way is a ring from here
      tc::wait_for_copies(full, depth, min(slices, s + depth));
      break;
    }
    const float* base = ring + b * stage_floats;
    const float* w = base + col * PITCH;
    constexpr int AHEAD = 4;  // pieces of four k in registers while as many are multiplied
    const int kn = min(SLICE, K - s * SLICE);
    float4 w4[2][AHEAD][CPT], x4[2][AHEAD][RPT];
    auto read = [&](int f, int k0) {
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
#pragma unroll
        for (int c = 0; c < CPT; ++c) w4[f][i][c] = *reinterpret_cast<const float4*>(w + 16 * c * PITCH + k0 + 4 * i);
#pragma unroll
        for (int r = 0; r < RPT; ++r) x4[f][i][r] = *reinterpret_cast<const float4*>(base + xat[r] + k0 + 4 * i);
      }
    };
    auto multiply = [&](int f, int i) {
#pragma unroll
      for (int r = 0; r < RPT; ++r)
#pragma unroll
        for (int c = 0; c < CPT; ++c) acc[r][c] = fmaf(x4[f][i][r].x, w4[f][i][c].x, acc[r][c]);
#pragma unroll
      for (int r = 0; r < RPT; ++r)
#pragma unroll
        for (int c = 0; c < CPT; ++c) acc[r][c] = fmaf(x4[f][i][r].y, w4[f][i][c].y, acc[r][c]);
#pragma unroll
      for (int r = 0; r < RPT; ++r)
#pragma unroll
        for (int c = 0; c < CPT; ++c) acc[r][c] = fmaf(x4[f][i][r].z, w4[f][i][c].z, acc[r][c]);
#pragma unroll
      for (int r = 0; r < RPT; ++r)
#pragma unroll
        for (int c = 0; c < CPT; ++c) acc[r][c] = fmaf(x4[f][i][r].w, w4[f][i][c].w, acc[r][c]);
    };
    if (kn == SLICE) {
      read(0, 0);
#pragma unroll
      for (int p = 0; p < SLICE / (4 * AHEAD); ++p) {
        if (p + 1 < SLICE / (4 * AHEAD)) read((p + 1) & 1, (p + 1) * 4 * AHEAD);
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) multiply(p & 1, i);
      }
    } else {
      for (int k = 0; k < kn; k += 4) {
#pragma unroll
        for (int c = 0; c < CPT; ++c) w4[0][0][c] = *reinterpret_cast<const float4*>(w + 16 * c * PITCH + k);
#pragma unroll
        for (int r = 0; r < RPT; ++r) x4[0][0][r] = *reinterpret_cast<const float4*>(base + xat[r] + k);
        multiply(0, 0);
      }
    }
    __syncwarp();
    if (lane == 0) tc::mbar_arrive(free_ + b);
    if (++b == depth) { b = 0; ++round; }
  }
  if (!here && lane == 0 && error) atomicExch(error, 20);
  if constexpr (More::ON) {
    more.wait();
    int n[CPT];
#pragma unroll
    for (int c = 0; c < CPT; ++c) n[c] = n0 + col + 16 * c < N ? n0 + col + 16 * c : -1;
    more.add(acc, row0, M, n);
  }
#pragma unroll
  for (int r = 0; r < RPT; ++r)
#pragma unroll
    for (int c = 0; c < CPT; ++c)
      if (row0 + r < M && n0 + col + 16 * c < N) C[(size_t)(row0 + r) * ldc + n0 + col + 16 * c] = here ? acc[r][c] : NAN;
}

template <int RPT, int CPT, int SLICE, typename More>
int launch_few(float* C, const float* A, const float* W, int M, int N, int K, int lda, int ldw, int ldc, int* error, const More& more, cudaStream_t stream) {
  constexpr size_t per_row = (SLICE + 4) * sizeof(float);
  const size_t stage = (16 * CPT + M) * per_row;  // 17 to 50 KB
  const int blocks = (N + 16 * CPT - 1) / (16 * CPT);
  // Two slices of the ring leave an SM more blocks than three, three cover more of a slice's way. Where a thread has one output, what
  // decides is how many blocks the SMs take in full rounds (three rows of K 2,560, two slices and three: N of 2,560 17.8 and 16.4 us, 6,144
  // 20.3 and 19.0, 8,192 22.6 and 29.3, 12,288 (K 4,096) 51.6 and 44.3, 19,456 43.0 and 44.0, 151,936 239 and 256). Two rows by two columns are
  // bound by the multiplying warps' own reads, which only other blocks cover: two slices at every size measured, where three were within 2 %
  // or worse (K 2,560, two and three: five rows in slices of 128, N of 151,936 277 and 365 us; sixteen rows in slices of 256, one
  // block an SM with three, 19,456 79 and 108, 151,936 438 and 698; twelve of 9,728 48 and 61).
  auto rounds = [&](int depth) {
    const long long held = max(1LL, (long long)(227 * 1024 / (FEW_BARS + depth * stage + 1024)));
    return (blocks + 148 * held - 1) / (148 * held) * held;
  };
  const int depth = RPT == 1 && rounds(3) < rounds(2) ? 3 : 2;
  // always the most that a call may need: another thread may be about to launch with more rows than this one
  cudaError_t e = cudaFuncSetAttribute(gemm_f32_few_kernel<RPT, CPT, SLICE, More>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       (int)(FEW_BARS + FEW_MAX_DEPTH * (16 * CPT + 8 * RPT) * per_row));
  if (e != cudaSuccess) return (int)e;
  const int readers = (M + 2 * RPT - 1) / (2 * RPT);
  if constexpr (More::ON)
    return (int)launch_pdl(gemm_f32_few_kernel<RPT, CPT, SLICE, More>, dim3(blocks), dim3(32 * (readers + 1)), FEW_BARS + depth * stage, stream, C, A, W, M, N, K,
                           lda, ldw, ldc, depth, error, more);
  gemm_f32_few_kernel<RPT, CPT, SLICE, More><<<blocks, 32 * (readers + 1), FEW_BARS + depth * stage, stream>>>(
      C, A, W, M, N, K, lda, ldw, ldc, depth, error, more);
  KRK_CHECK_LAUNCH();
  return 0;
}

// M <= 16, 16-byte rows and addresses.
template <typename More>
int launch_f32_few(float* C, const float* A, const float* W, int M, int N, int K, int lda, int ldw, int ldc, int* error, const More& more, cudaStream_t stream) {
  // 16 rows: 79 us of 19,456 x 2,560 and 161 by the tiles below, 438 and 647 of 151,936 x 2,560, 2.5 and 4.0 of 128 x 64.
  // One row of one column a thread reads most of shared memory for a multiply-add and has the most blocks; from five rows
  // on the reads bound it where there are columns enough (eight rows, two by two in slices of 128 and one by one: N of 19,456
  // 45 and 57 us, 151,936 283 and 366; 8,192 27 and 22; five rows 44 and 48, 277 and 284; 12,288 31 and 28). Beyond eight rows two by
  // two always: in slices of 128 to 12 rows of many columns (nine rows: N of 12,288 32 and 41, 151,936 322 and 399; 8,192 28 and 22;
  // sixteen 437 and 438, but 89 and 79 of 19,456).
  if (M <= 8 && (M < 5 || N < 16384)) return launch_few<1, 1, 256>(C, A, W, M, N, K, lda, ldw, ldc, error, more, stream);
  if (M <= 8 || (M <= 12 && N >= 12288)) return launch_few<2, 2, 128>(C, A, W, M, N, K, lda, ldw, ldc, error, more, stream);
  return launch_few<2, 2, 256>(C, A, W, M, N, K, lda, ldw, ldc, error, more, stream);
}

}  // namespace
