// Tiles of attention on the warp-level tensor cores (mma.sync m16n8k16): a page of keys or values in shared memory, Q K^T, the
// online softmax and P V of 16 rows. For the sources that are compiled once per head size, -DKRK_HEAD_DIM=<D>, D a multiple
// of 16 up to 256; included inside an anonymous namespace.
#pragma once

constexpr int D = KRK_HEAD_DIM;
constexpr int DP = D + 8;            // shared-memory row pitch (elements): 16 bytes of padding
constexpr int KSTEPS = D / 16;       // k-steps of Q.K^T
constexpr int DTILES = D / 8;        // n-tiles of P.V
constexpr int THREADS = 128;
// A page of keys or values in shared memory. Where a row is a power-of-two number (at least eight) of
// 16-byte pieces, rows are packed and piece c of key k sits at piece c ^ (k & 7), which spreads the eight
// rows of an ldmatrix over all banks without padding; other head sizes pad each row by 16 bytes instead.
constexpr bool KV_SWIZZLE = (D == 64 || D == 128 || D == 256);
constexpr int KVP = KV_SWIZZLE ? D : DP;  // row pitch of a page in shared memory (elements)
constexpr int TILE_ELEMS = KRK_PAGE * KVP;
__device__ __forceinline__ int kv_off(int key, int piece) {
  return key * KVP + ((KV_SWIZZLE ? (piece ^ (key & 7)) : piece) << 3);
}
// The same page as TMA writes it with the 128-byte swizzle: D / 64 sub-tiles of [64 keys][128 bytes], piece c of
// key k of a sub-tile at piece c ^ (k & 7). Head sizes that are multiples of 64 only.
constexpr bool TMA_PAGES = (D % 64 == 0);
constexpr int SUB_ELEMS = KRK_PAGE * 64;  // elements of one sub-tile (8 KB)
template <bool TMA>
__device__ __forceinline__ int page_off(int key, int piece) {
  if (TMA) return (piece >> 3) * SUB_ELEMS + key * 64 + (((piece & 7) ^ (key & 7)) << 3);
  return kv_off(key, piece);
}
constexpr float LOG2E = 1.4426950408889634f;

constexpr size_t PAGE_SMEM = (size_t)2 * 2 * TILE_ELEMS * sizeof(bf16);  // two stages of a page of keys and one of values

// Copy one page [64][D] of one kv head to shared memory [64][DP], all threads of the block.
__device__ __forceinline__ void load_page(bf16* dst, const bf16* __restrict__ src) {
  constexpr int CHUNKS = KRK_PAGE * (D / 8);
  for (int i = threadIdx.x; i < CHUNKS; i += THREADS) {
    const int key = i / (D / 8), ch = i % (D / 8);
    cp_async_16(dst + kv_off(key, ch), src + key * D + ch * 8);
  }
}

// S[16 x (8*NTILES)] = Q[16 x D] . K^T for keys key0 .. key0 + 8*NTILES - 1 of the tile in shared memory.
template <int NTILES, bool TMA = false>
__device__ __forceinline__ void qk_tile(float (&s)[NTILES][4], const uint32_t (&qf)[KSTEPS][4], const bf16* ks, int key0,
                                        int lane) {
  // even and odd k-steps accumulate apart and are added at the end: two chains of KSTEPS / 2 dependent MMAs
  // per n-tile instead of one of KSTEPS
  float odd[NTILES][4];
#pragma unroll
  for (int n = 0; n < NTILES; ++n)
#pragma unroll
    for (int c = 0; c < 4; ++c) s[n][c] = odd[n][c] = 0.f;
#pragma unroll
  for (int kk = 0; kk < KSTEPS; ++kk) {
#pragma unroll
    for (int n = 0; n < NTILES; n += 2) {
      uint32_t b0, b1, b2, b3;
      const bf16* p = ks + page_off<TMA>(key0 + n * 8 + ((lane >> 4) << 3) + (lane & 7), kk * 2 + ((lane >> 3) & 1));
      ldmatrix_x4(b0, b1, b2, b3, p);
      if (kk & 1) {
        mma_bf16_16816(odd[n], qf[kk][0], qf[kk][1], qf[kk][2], qf[kk][3], b0, b1);
        mma_bf16_16816(odd[n + 1], qf[kk][0], qf[kk][1], qf[kk][2], qf[kk][3], b2, b3);
      } else {
        mma_bf16_16816(s[n], qf[kk][0], qf[kk][1], qf[kk][2], qf[kk][3], b0, b1);
        mma_bf16_16816(s[n + 1], qf[kk][0], qf[kk][1], qf[kk][2], qf[kk][3], b2, b3);
      }
    }
  }
#pragma unroll
  for (int n = 0; n < NTILES; ++n)
#pragma unroll
    for (int c = 0; c < 4; ++c) s[n][c] += odd[n][c];
}

// O[16 x D] += P[16 x (8*NTILES)] . V for the same keys; p holds probabilities (float) in S's layout.
template <int NTILES, bool TMA = false>
__device__ __forceinline__ void pv_tile(float (&o)[DTILES][4], const float (&p)[NTILES][4], const bf16* vs, int key0,
                                        int lane) {
#pragma unroll
  for (int kk = 0; kk < NTILES / 2; ++kk) {  // 16 keys per step
    const uint32_t a0 = pack_bf16x2(p[2 * kk][0], p[2 * kk][1]);
    const uint32_t a1 = pack_bf16x2(p[2 * kk][2], p[2 * kk][3]);
    const uint32_t a2 = pack_bf16x2(p[2 * kk + 1][0], p[2 * kk + 1][1]);
    const uint32_t a3 = pack_bf16x2(p[2 * kk + 1][2], p[2 * kk + 1][3]);
#pragma unroll
    for (int n = 0; n < DTILES; n += 2) {
      uint32_t b0, b1, b2, b3;
      const bf16* q = vs + page_off<TMA>(key0 + kk * 16 + (lane & 7) + ((lane >> 3) & 1) * 8, n + (lane >> 4));
      ldmatrix_x4_trans(b0, b1, b2, b3, q);
      mma_bf16_16816(o[n], a0, a1, a2, a3, b0, b1);
      mma_bf16_16816(o[n + 1], a0, a1, a2, a3, b2, b3);
    }
  }
}

// The same with the probabilities kept to about 16 bits of mantissa: p = hi + lo with both halves bfloat16, two
// MMAs per fragment of V. For models whose softmax weights are 32-bit quantities: what is lost is below
// 2^-16 of a weight, the order of the float32 exponential's own error.
template <int NTILES>
__device__ __forceinline__ void pv_tile_wide(float (&o)[DTILES][4], const float (&p)[NTILES][4], const bf16* vs, int key0,
                                             int lane) {
#pragma unroll
  for (int kk = 0; kk < NTILES / 2; ++kk) {
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int f = 0; f < 4; ++f) {
      const float x = p[2 * kk + (f >> 1)][2 * (f & 1)], y = p[2 * kk + (f >> 1)][2 * (f & 1) + 1];
      const float xh = __bfloat162float(__float2bfloat16_rn(x)), yh = __bfloat162float(__float2bfloat16_rn(y));
      hi[f] = pack_bf16x2(xh, yh);
      lo[f] = pack_bf16x2(x - xh, y - yh);
    }
#pragma unroll
    for (int n = 0; n < DTILES; n += 2) {
      uint32_t b0, b1, b2, b3;
      const bf16* q = vs + page_off<false>(key0 + kk * 16 + (lane & 7) + ((lane >> 3) & 1) * 8, n + (lane >> 4));
      ldmatrix_x4_trans(b0, b1, b2, b3, q);
      mma_bf16_16816(o[n], hi[0], hi[1], hi[2], hi[3], b0, b1);
      mma_bf16_16816(o[n], lo[0], lo[1], lo[2], lo[3], b0, b1);
      mma_bf16_16816(o[n + 1], hi[0], hi[1], hi[2], hi[3], b2, b3);
      mma_bf16_16816(o[n + 1], lo[0], lo[1], lo[2], lo[3], b2, b3);
    }
  }
}

// Load the A fragments of one 16-row tile of queries; row r of the tile is at qrow[r half] (null: zero row).
__device__ __forceinline__ void load_q(uint32_t (&qf)[KSTEPS][4], const bf16* q_lo, const bf16* q_hi, int lane) {
  const int t = lane & 3;
#pragma unroll
  for (int kk = 0; kk < KSTEPS; ++kk) {
    const int d = kk * 16 + 2 * t;
    qf[kk][0] = q_lo ? *reinterpret_cast<const uint32_t*>(q_lo + d) : 0u;
    qf[kk][1] = q_hi ? *reinterpret_cast<const uint32_t*>(q_hi + d) : 0u;
    qf[kk][2] = q_lo ? *reinterpret_cast<const uint32_t*>(q_lo + d + 8) : 0u;
    qf[kk][3] = q_hi ? *reinterpret_cast<const uint32_t*>(q_hi + d + 8) : 0u;
  }
}

__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// One online-softmax update of a thread's two rows over NTILES*8 keys. s is in log2
// units already (scaled by scale*log2(e)) and masked with -inf where invisible.
template <int NTILES>
__device__ __forceinline__ void softmax_update(float (&s)[NTILES][4], float (&m)[2], float (&l)[2], float (&o)[DTILES][4]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float mx = -INFINITY;
#pragma unroll
    for (int n = 0; n < NTILES; ++n) mx = fmaxf(mx, fmaxf(s[n][2 * h], s[n][2 * h + 1]));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    const float m_new = fmaxf(m[h], mx);
    const float m_safe = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = fast_exp2(m[h] - m_safe);
    float sum = 0.f;
#pragma unroll
    for (int n = 0; n < NTILES; ++n) {
      s[n][2 * h] = fast_exp2(s[n][2 * h] - m_safe);
      s[n][2 * h + 1] = fast_exp2(s[n][2 * h + 1] - m_safe);
      sum += s[n][2 * h] + s[n][2 * h + 1];
    }
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
    l[h] = l[h] * alpha + sum;
    m[h] = m_new;
#pragma unroll
    for (int n = 0; n < DTILES; ++n) {
      o[n][2 * h] *= alpha;
      o[n][2 * h + 1] *= alpha;
    }
  }
}
