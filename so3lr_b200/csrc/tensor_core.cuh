// Building blocks of the dense tcgen05 kernels (dense.cu): mbarriers with bounded
// waits, TMA tile loads, shared-memory and instruction descriptors, MMAs of a CTA
// pair and TMEM reads.
//
// A CTA pair (cluster of 2, cta_group::2) computes one tile of 256 rows: each
// CTA's shared memory holds its own 128 rows of A and half of the rows of B, its
// TMEM its own 128 rows of the result. The even CTA (the leader) issues the MMAs
// for both. Each CTA fetches its own part of a tile, from this GPU's memory, and
// completes it on the leader's barrier.
#pragma once

#include <cuda.h>

#include <cstdint>

namespace so3lr_b200 {
namespace tc {

constexpr long long kWaitCycles = 4000000000LL;  // about 2 s at 1.9 GHz
constexpr long long kPolled = 20000;             // limits below it: a blocking try alone takes 8,000 cycles

__device__ __forceinline__ uint32_t smem_u32(const volatile void *p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(const_cast<const void *>(p)));
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_index() {
  uint32_t i;
  asm("mov.u32 %0, %%clusterid.x;" : "=r"(i));
  return i;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t n;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(n));
  return n;
}
// a 32-bit shared variable of another block of the cluster
template <class T>
__device__ __forceinline__ T load_of_rank(const volatile T *own, uint32_t rank) {
  uint32_t at, bits;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(own)), "r"(rank));
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(bits) : "r"(at) : "memory");
  return reinterpret_cast<const T &>(bits);
}
__device__ __forceinline__ void store_of_rank(volatile int *own, uint32_t rank, int v) {
  uint32_t at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(own)), "r"(rank));
  asm volatile("st.volatile.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(v) : "memory");
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// the address of the leader's copy of a shared variable
__device__ __forceinline__ uint32_t at_leader(uint32_t addr) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
  return r;
}

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count));
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.release.cta.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes)
               : "memory");
}
// `bytes` that a barrier expects and that will not be copied (a shared::cluster address)
__device__ __forceinline__ void mbar_complete_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.complete_tx.relaxed.cluster.shared::cluster.b64 [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// arrive on a barrier of either CTA of the pair (a shared::cluster address). It hands
// over TMEM, which the tcgen05 fences order, and no memory: a cluster-wide release
// would wait for every global store of the warp (a sixth of the epilogue's time).
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
      " selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(done)
      : "r"(bar), "r"(parity)
      : "memory");
  return done != 0;
}
// the same, or (polled) without blocking. Two predicated instructions: it stands in every wait, and
// its code's length shows in small products (300 rows through the 256 x 1024 block 12.53 us, with
// a branch 12.60, with a call 13.17).
__device__ __forceinline__ bool mbar_try_or_test(uint32_t bar, uint32_t parity, bool polled) {
  uint32_t done;
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.u32 q, %3, 0;\n"
      " @!q mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
      " @q mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n"
      " selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(done)
      : "r"(bar), "r"(parity), "r"(uint32_t(polled))
      : "memory");
  return done != 0;
}
// Waits for the phase of the given parity, about `limit` cycles at most; false (with
// *abort_flag = mark and *err = where) when it gives up or another thread of the CTA
// already gave up.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int *abort_flag, int *err, int where,
                                          long long limit = kWaitCycles, int mark = 1) {
  const bool polled = limit < kPolled;
  if (mbar_try_or_test(bar, parity, polled)) return true;
  const long long t0 = clock64();
  while (!mbar_try_or_test(bar, parity, polled)) {
    if (*abort_flag) return false;
    if (clock64() - t0 > limit) {
      *abort_flag = mark;
      *reinterpret_cast<volatile int *>(err) = where;
      return false;
    }
  }
  return true;
}
// After a wait that gave up: waits for what is still under way into this block's
// memory, whoever gave up, until kWaitCycles after t0.
__device__ __forceinline__ void mbar_settle(uint32_t bar, uint32_t parity, long long t0) {
  while (!mbar_try(bar, parity) && clock64() - t0 < kWaitCycles) {
  }
}

// `bytes` (a multiple of 16) from 16-byte aligned global memory, completed on `bar`
__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// One box of a 2-D tensor map into this CTA's shared memory; `bar` may be the
// peer CTA's barrier. x is a multiple of 16 bytes; out-of-range elements read 0.
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap *map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, "
      "%4}], [%2];" ::"r"(dst),
      "l"(map), "r"(bar), "r"(x), "r"(y)
      : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap *map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

// Shared-memory operand descriptors, 128-byte swizzle, tiles on 1024-byte
// boundaries. K-major: rows of 128 bytes along K, 8-row groups 1024 bytes apart; a
// K step of 32 bytes advances the start address by 32. MN-major: rows of 64
// elements along M/N, one row per k, 8-k groups 1024 bytes apart, the next 64 of
// M/N `lbo` bytes further; a K step of 16 advances the start address by 2048.
__device__ __forceinline__ uint64_t desc_k(uint32_t saddr) {
  return uint64_t((saddr >> 4) & 0x3fff) | (uint64_t(1) << 16) | (uint64_t(1024 >> 4) << 32) | (uint64_t(1) << 46) |
         (uint64_t(2) << 61);
}
__device__ __forceinline__ uint64_t desc_mn(uint32_t saddr, uint32_t lbo) {
  return uint64_t((saddr >> 4) & 0x3fff) | (uint64_t(lbo >> 4) << 16) | (uint64_t(1024 >> 4) << 32) |
         (uint64_t(1) << 46) | (uint64_t(2) << 61);
}
// Instruction descriptor: d, a, b formats; operands MN-major or not; N columns, 256 rows.
constexpr uint32_t idesc(uint32_t d, uint32_t ab, bool a_mn, bool b_mn, int n) {
  return (d << 4) | (ab << 7) | (ab << 10) | (uint32_t(a_mn) << 15) | (uint32_t(b_mn) << 16) |
         (uint32_t(n >> 3) << 17) | (uint32_t(256 >> 4) << 24);
}
template <bool INT8>
__device__ __forceinline__ void mma(uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t id, bool accumulate) {
  if (INT8)
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n}\n" ::"r"(d_tmem),
        "l"(a), "l"(b), "r"(id), "r"(uint32_t(accumulate)));
  else
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d_tmem),
        "l"(a), "l"(b), "r"(id), "r"(uint32_t(accumulate)));
}
// completion of the MMAs issued so far, on the barrier at this offset of both CTAs
__device__ __forceinline__ void commit_pair(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
      "h"(uint16_t(3))
      : "memory");
}
// 32 consecutive 32-bit columns of this warp's 32 TMEM lanes (complete after wait_ld)
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,"
      "%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void wait_ld(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]),
                 "+r"(r[15])::"memory");
}
// waits for this thread's TMEM reads; the registers are operands so that nothing
// that uses them moves ahead of the wait
__device__ __forceinline__ void wait_ld(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]),
                 "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]),
                 "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]),
                 "+r"(r[29]), "+r"(r[30]), "+r"(r[31])::"memory");
}

}  // namespace tc
}  // namespace so3lr_b200
