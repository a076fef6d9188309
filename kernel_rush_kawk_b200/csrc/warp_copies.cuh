// Copies by TMA, and what their barriers are told, asked for by a whole warp.
#pragma once

#include "tcgen05.cuh"

namespace tc {

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
__device__ __forceinline__ void tma_load_2d_warp(uint32_t smem_dst, const CUtensorMap* map, uint32_t bar, int x, int y) {
  asm volatile(
      "{\n.reg .pred q;\n"
      "elect.sync _|q, 0xffffffff;\n"
      "@q cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];\n}"
      ::"r"(smem_dst), "l"(map), "r"(bar), "r"(x), "r"(y)
      : "memory");
}
__device__ __forceinline__ void mbar_expect_tx_warp(uint32_t bar, uint32_t bytes) {
  asm volatile(
      "{\n.reg .pred q;\n"
      "elect.sync _|q, 0xffffffff;\n"
      "@q mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n}"
      ::"r"(bar), "r"(bytes)
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
