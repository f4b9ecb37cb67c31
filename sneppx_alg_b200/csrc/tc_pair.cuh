// What the kernels on a pair of CTAs (`cta_group::2`) share: a cluster of two SMs owns one tile of 256 rows, each CTA stages its half of both operands,
// the even CTA issues the MMAs, each CTA's TMEM holds the accumulator rows of its half of A.
#pragma once
#include "tc_common.cuh"

namespace sx {

// Tile t of a persistent kernel: groups of eight row blocks go through all column blocks together.
__device__ __forceinline__ void tile_coords(int t, int m_blks, int n_blks, int& b, int& m_blk, int& n_blk) {
  const int per_batch = m_blks * n_blks;
  b = t / per_batch;
  int r = t - b * per_batch;
  constexpr int GM = 8;
  const int group_sz = GM * n_blks;
  const int g = r / group_sz;
  const int first_m = g * GM;
  const int gsz = min(GM, m_blks - first_m);
  const int rr = r - g * group_sz;
  m_blk = first_m + rr % gsz;
  n_blk = rr / gsz;
}

constexpr uint32_t PEER_MASK = 0xFEFFFFFFu;  // clears the CTA-rank bit of a shared::cluster address: the even CTA's copy

__device__ __forceinline__ uint32_t cluster_ctarank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void tma2_load_3d(void* dst, const CUtensorMap* m, uint32_t bar_cluster_addr, int c0, int c1,
                                             int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(m)), "r"(bar_cluster_addr), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}
__device__ __forceinline__ void tma2_load_4d(void* dst, const CUtensorMap* m, uint32_t bar_cluster_addr, int c0, int c1,
                                             int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
      ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(m)), "r"(bar_cluster_addr), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}
__device__ __forceinline__ void umma2_f16_ss(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                             uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5, %5, %5, %5, %5}, p;\n}\n" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(0u)
      : "memory");
}
// Arrives (once the MMAs issued so far have executed) on the barrier at this offset in BOTH CTAs of the pair.
__device__ __forceinline__ void umma2_commit_pair(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"((uint16_t)3)
      : "memory");
}
// Hands an accumulator back to the even CTA's MMA thread. All that it says is that this warp's tcgen05.ld are done, which tcgen05.wait::ld has seen to in
// each lane, so it is relaxed: a release at cluster scope would first wait for the warp's stores to global memory (4096 x 32000 logits of width 512:
// tiles of the loss 115 -> 94 us forward and 134 -> 117 backward).
__device__ __forceinline__ void mbar_arrive_even_cta(uint64_t* bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(smem_u32(bar) & PEER_MASK) : "memory");
}

}  // namespace sx
