// Copies by TMA, and what their barriers are told, asked for by a whole warp.
#pragma once

#include "tcgen05.cuh"

namespace tc {

// mbar_wait for long waits: the hardware may keep the thread asleep for up to 4 us a try, so that who has nothing to do draws little power.
__device__ __forceinline__ bool mbar_wait_long(uint64_t* bar, uint32_t parity, unsigned long long limit_ns = WAIT_LIMIT_NS) {
  const uint32_t addr = smem_u32(bar);
  unsigned long long t0 = 0;
  for (;;) {
    uint32_t done;
    asm volatile(
        "{\n.reg .pred p;\n"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n"
        "selp.u32 %0, 1, 0, p;\n}"
        : "=r"(done)
        : "r"(addr), "r"(parity), "r"(4000u)
        : "memory");
    if (done) return true;
    const unsigned long long now = global_ns();
    if (t0 == 0) t0 = now;
    else if (now - t0 > limit_ns) return false;
  }
}

// Asked for by a whole warp, one lane of which does it (see umma_bf16_warp). In a single lane's branch a block of k of the first factor took some
// 700 clocks, whatever was loaded.
__device__ __forceinline__ void tma_load_2d_pair_warp(uint32_t smem_dst, const CUtensorMap* map, uint32_t cluster_bar, int x, int y) {
  asm volatile(
      "{\n.reg .pred q;\n"
      "elect.sync _|q, 0xffffffff;\n"
      "@q cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];\n}"
      ::"r"(smem_dst), "l"(map), "r"(cluster_bar), "r"(x), "r"(y)
      : "memory");
}
__device__ __forceinline__ void tma_load_3d_pair_warp(uint32_t smem_dst, const CUtensorMap* map, uint32_t cluster_bar, int x, int y, int z) {
  asm volatile(
      "{\n.reg .pred q;\n"
      "elect.sync _|q, 0xffffffff;\n"
      "@q cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];\n}"
      ::"r"(smem_dst), "l"(map), "r"(cluster_bar), "r"(x), "r"(y), "r"(z)
      : "memory");
}
__device__ __forceinline__ void tma_load_4d_pair_warp(uint32_t smem_dst, const CUtensorMap* map, uint32_t cluster_bar, int x, int y, int z, int u) {
  asm volatile(
      "{\n.reg .pred q;\n"
      "elect.sync _|q, 0xffffffff;\n"
      "@q cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];\n}"
      ::"r"(smem_dst), "l"(map), "r"(cluster_bar), "r"(x), "r"(y), "r"(z), "r"(u)
      : "memory");
}
// Two copies that one barrier counts, and the barrier's bytes.
__device__ __forceinline__ void two_loads_warp(uint32_t to0, const CUtensorMap* map0, int x0, int y0, uint32_t to1, const CUtensorMap* map1, int x1, int y1, uint32_t bar,
                                               uint32_t bytes) {
  asm volatile(
      "{\n.reg .pred q;\n"
      "elect.sync _|q, 0xffffffff;\n"
      "@q mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n"
      "@q cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%2], [%3, {%4, %5}], [%0];\n"
      "@q cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%6], [%7, {%8, %9}], [%0];\n}"
      ::"r"(bar), "r"(bytes), "r"(to0), "l"(map0), "r"(x0), "r"(y0), "r"(to1), "l"(map1), "r"(x1), "r"(y1)
      : "memory");
}
// Leaves a word for who waits on the barrier, and says how many bytes it waits for.
__device__ __forceinline__ void expect_with_word_warp(uint32_t bar, uint32_t bytes, uint32_t word_at, int word) {
  asm volatile(
      "{\n.reg .pred q;\n"
      "elect.sync _|q, 0xffffffff;\n"
      "@q st.shared.u32 [%2], %3;\n"
      "@q mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n}"
      ::"r"(bar), "r"(bytes), "r"(word_at), "r"(word)
      : "memory");
}

}  // namespace tc
