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
//
// A stage of a pair of blocks: the two copies that one of them brings, of DIMS and of two dimensions, both counted on the first block's barrier; the first block
// (`expects`) leaves a word for who waits there and says how many bytes both bring. All in one election, which
// takes 59 clocks; with one for each, and the wait for the first factor asked in every turn, an adapter's stage took its producer 762 clocks, now some 600 (of 64
// adapters beside gate and up of 2,560 x 19,456, 64 rows: 84 -> 78 us).
struct PairStage {
  uint32_t bar, own_bar, bytes, word_at;  // the first block's barrier, as both name it and as it does itself
  uint32_t expects;
};
#define KRK_STAGE_BEGIN                                                  \
  "{\n.reg .pred q, r;\n"                                                \
  "elect.sync _|q, 0xffffffff;\n"                                        \
  "setp.ne.and.b32 r, %4, 0, q;\n"                                       \
  "@r st.shared.u32 [%3], %5;\n"                                         \
  "@r mbarrier.arrive.expect_tx.shared::cta.b64 _, [%1], %2;\n"
#define KRK_STAGE_SECOND "@q cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%8], [%9, {%10, %11}], [%0];\n"
#define KRK_STAGE_ARGS                                                                                                                                        \
  "r"(s.bar), "r"(s.own_bar), "r"(s.bytes), "r"(s.word_at), "r"(s.expects), "r"(word), "r"(to0), "l"(map0), "r"(to1), "l"(map1), "r"(x1), "r"(y1)
__device__ __forceinline__ void stage_2d_2d_warp(const PairStage& s, int word, uint32_t to0, const CUtensorMap* map0, int x0, int y0, uint32_t to1, const CUtensorMap* map1, int x1,
                                                 int y1) {
  asm volatile(KRK_STAGE_BEGIN
               "@q cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%6], [%7, {%12, %13}], [%0];\n" KRK_STAGE_SECOND "}"
               ::KRK_STAGE_ARGS, "r"(x0), "r"(y0)
               : "memory");
}
__device__ __forceinline__ void stage_3d_2d_warp(const PairStage& s, int word, uint32_t to0, const CUtensorMap* map0, int x0, int y0, int z0, uint32_t to1, const CUtensorMap* map1,
                                                 int x1, int y1) {
  asm volatile(KRK_STAGE_BEGIN
               "@q cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%6], [%7, {%12, %13, %14}], [%0];\n" KRK_STAGE_SECOND "}"
               ::KRK_STAGE_ARGS, "r"(x0), "r"(y0), "r"(z0)
               : "memory");
}
__device__ __forceinline__ void stage_4d_2d_warp(const PairStage& s, int word, uint32_t to0, const CUtensorMap* map0, int x0, int y0, int z0, int u0, uint32_t to1,
                                                 const CUtensorMap* map1, int x1, int y1) {
  asm volatile(KRK_STAGE_BEGIN
               "@q cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%6], [%7, {%12, %13, %14, %15}], [%0];\n" KRK_STAGE_SECOND "}"
               ::KRK_STAGE_ARGS, "r"(x0), "r"(y0), "r"(z0), "r"(u0)
               : "memory");
}
#undef KRK_STAGE_BEGIN
#undef KRK_STAGE_SECOND
#undef KRK_STAGE_ARGS
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
}  // namespace tc
