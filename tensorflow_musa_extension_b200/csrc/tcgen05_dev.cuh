// Device helpers of the matrix-product kernels: mbarriers with bounded waits, TMA
// tile copies, tensor memory and the tcgen05 matrix instructions (PTX ISA 8.6+).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace musa_b200 {

__device__ __forceinline__ uint32_t SmemAddr(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

// ---- mbarriers.  Addresses are shared::cta offsets, which name the CTA's own
// barrier in the cluster window too; MapToCta gives the same barrier of a peer.
__device__ __forceinline__ void BarInit(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void BarInitFence() {
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
}
__device__ __forceinline__ void BarExpect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ uint32_t MapToCta(uint32_t addr, uint32_t rank) {
  uint32_t out;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(out) : "r"(addr), "r"(rank));
  return out;
}
__device__ __forceinline__ void BarArriveCluster(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr)
               : "memory");
}
__device__ __forceinline__ bool BarTry(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n.reg .pred p;\n"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
      "selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(done)
      : "r"(bar), "r"(parity)
      : "memory");
  return done != 0;
}

// Waits give up after about two seconds, far beyond any launch: `give_up` (shared
// memory of the CTA) tells the CTA's other roles, `status` (global) the host.  A role
// that sees false leaves its loop; LeaveInFlight then lets the copies and matrix
// instructions already issued land before the CTA frees what they write.
constexpr long long kWaitCycles = 4000000000LL;

// A whole warp waits, with one answer for it: the loops around the waits stay uniform, so that
// their addresses and descriptors live in the uniform registers that the TMA and matrix
// instructions read (with one lane looping alone a stage took 650 cycles, whatever the tile).
__device__ __noinline__ bool BarWaitSlow(uint32_t bar, uint32_t parity, volatile int* give_up,
                                         int* status) {
  const long long begin = clock64();
  for (;;) {
    const bool late = clock64() - begin > kWaitCycles;
    if (__all_sync(0xffffffffu, BarTry(bar, parity))) return true;
    if (__any_sync(0xffffffffu, late || *give_up != 0)) {
      if (late) {
        *give_up = 1;
        atomicExch(status, 1);
      }
      return false;
    }
  }
}
__device__ __forceinline__ bool BarWait(uint32_t bar, uint32_t parity, volatile int* give_up,
                                        int* status) {
  if (__all_sync(0xffffffffu, BarTry(bar, parity))) return true;
  return __all_sync(0xffffffffu, BarWaitSlow(bar, parity, give_up, status));
}
// One lane of a converged warp.
__device__ __forceinline__ bool ElectLane() {
  uint32_t yes;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}\n"
               : "=r"(yes));
  return yes != 0;
}
__device__ __forceinline__ void LeaveInFlight() {
  for (int i = 0; i < 2000; ++i) __nanosleep(1000);
}

// ---- TMA.  `bar` of a load may be a cluster address.  With kPair the barrier may lie in
// the other CTA of the pair.
template <bool kPair>
__device__ __forceinline__ void TmaLoad(uint32_t dst, const CUtensorMap* map, int c0, int c1,
                                        uint32_t bar) {
  if constexpr (kPair) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        ".cta_group::2 [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(map), "r"(c0), "r"(c1), "r"(bar)
        : "memory");
  } else {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(map), "r"(c0), "r"(c1), "r"(bar)
        : "memory");
  }
}
__device__ __forceinline__ void TmaStore(const CUtensorMap* map, int c0, int c1, uint32_t src) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];"
               ::"l"(map), "r"(c0), "r"(c1), "r"(src)
               : "memory");
}
__device__ __forceinline__ void TmaStoreCommit() {
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
template <int kPending>
__device__ __forceinline__ void TmaStoreWaitRead() {
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(kPending) : "memory");
}
__device__ __forceinline__ void TmaStoreWaitAll() {
  asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
}
__device__ __forceinline__ void FenceAsyncShared() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
// ---- Tensor memory: 128 lanes x 512 columns of 32 bits per SM.
template <int kGroup>
__device__ __forceinline__ void TmemAlloc(uint32_t smem_dst, uint32_t columns) {
  if constexpr (kGroup == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_dst),
                 "r"(columns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  } else {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_dst),
                 "r"(columns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
}
template <int kGroup>
__device__ __forceinline__ void TmemFree(uint32_t addr, uint32_t columns) {
  if constexpr (kGroup == 2) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr),
                 "r"(columns));
  } else {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr),
                 "r"(columns));
  }
}
__device__ __forceinline__ void TmemFenceBefore() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void TmemFenceAfter() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}

// 32 lanes (the warp's quarter of the tensor memory) x 16 / 32 columns.
__device__ __forceinline__ void TmemLoad(uint32_t addr, float (&v)[16]) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void TmemLoad(uint32_t addr, float (&v)[32]) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, "
      "%20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
        "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
        "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
// The registers of the loads above hold their values after this.
template <int kN>
__device__ __forceinline__ void TmemLoadWait(float (&v)[kN]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < kN; ++i) asm volatile("" : "+f"(v[i]));
}

// ---- Matrix instructions.  Operands lie in shared memory in tiles of 128-byte rows
// with the 128-byte swizzle, each 1024-byte aligned:
//   depth-major (the reduction is contiguous)  rows of the operand, 128 bytes of depth
//                          each; groups of eight rows are 1024 bytes apart
//   row-major  (the operand's rows are contiguous: a transposed operand)  blocks of 64
//                          operand rows x 64 depths; groups of eight depths are 1024
//                          bytes apart, blocks of 64 rows 8192
// Bits of the descriptor: address / 16 at 0, leading offset / 16 at 16, stride offset
// / 16 at 32, constant 1 at 46, swizzle 2 (128 bytes) at 61.
constexpr uint32_t kBlockBytes = 64 * 128;

__device__ __forceinline__ uint64_t OperandDesc(uint32_t addr, bool rows_contiguous) {
  const uint64_t lead = rows_contiguous ? kBlockBytes / 16 : 1;
  return (static_cast<uint64_t>(2) << 61) | (static_cast<uint64_t>(1) << 46) |
         (static_cast<uint64_t>(1024 / 16) << 32) | (lead << 16) |
         static_cast<uint64_t>((addr & 0x3ffff) >> 4);
}
// What one instruction's depth (32 bytes) adds to the descriptor.
__host__ __device__ constexpr uint32_t DepthStep(bool rows_contiguous) {
  return rows_contiguous ? 2048 / 16 : 32 / 16;
}

// Instruction descriptor: fp32 accumulator, operand types (kind::f16: 0 half, 1 bfloat16;
// kind::f8f6f4: 0 e4m3), transposition flags, n / 8 at 17, m / 16 at 24.
__host__ __device__ constexpr uint32_t InstructionDesc(int type, bool a_rows, bool b_rows, int m,
                                                       int n) {
  return (1u << 4) | (static_cast<uint32_t>(type) << 7) | (static_cast<uint32_t>(type) << 10) |
         (a_rows ? 1u << 15 : 0u) | (b_rows ? 1u << 16 : 0u) |
         (static_cast<uint32_t>(n / 8) << 17) | (static_cast<uint32_t>(m / 16) << 24);
}

template <int kGroup, bool kBytes>
__device__ __forceinline__ void Mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                    bool accumulate) {
  const uint32_t add = accumulate ? 1 : 0;
#define MUSA_MMA(GROUP, KIND)                                                              \
  asm volatile("{\n.reg .pred p;\nsetp.ne.u32 p, %4, 0;\n"                                 \
               "tcgen05.mma.cta_group::" GROUP ".kind::" KIND " [%0], %1, %2, %3, p;\n}\n" \
               ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(add)                              \
               : "memory")
  if constexpr (kGroup == 2) {
    if constexpr (kBytes) MUSA_MMA("2", "f8f6f4");
    else MUSA_MMA("2", "f16");
  } else {
    if constexpr (kBytes) MUSA_MMA("1", "f8f6f4");
    else MUSA_MMA("1", "f16");
  }
#undef MUSA_MMA
}

// An arrival on `bar` when all matrix instructions of this thread so far are done; of a
// pair: on the barrier at this offset in both CTAs.
template <int kGroup>
__device__ __forceinline__ void MmaCommit(uint32_t bar) {
  if constexpr (kGroup == 2) {
    const uint16_t both = 3;
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster"
        ".b64 [%0], %1;" ::"r"(bar),
        "h"(both)
        : "memory");
  } else {
    asm volatile(
        "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar)
        : "memory");
  }
}

}  // namespace musa_b200
