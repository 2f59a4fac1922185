// 5th-generation tensor core helpers (tcgen05, pairs of CTAs): descriptors of 128-byte-swizzled fp16 tiles in shared memory,
// tensor memory, and the instructions' wrappers.
#pragma once

#include "common.cuh"

namespace gmc {

// A matrix in two fp16 planes is stored in rows of 64 elements (128 bytes); the 16-byte chunk c of row r sits at chunk
// c ^ (r & 7). Eight rows of the first plane (1024 bytes) are followed by the same eight rows of the second one, so that any
// group of rows is one contiguous piece with both planes. The same tile is read along its rows (K contiguous: `k_major`)
// or across them (rows are the K axis: `mn_major`).
constexpr uint32_t kPlaneOffset = 1024, kGroupBytes = 2048;
__device__ __forceinline__ uint32_t swizzled_offset(int row, int chunk) {
    return uint32_t(row >> 3) * kGroupBytes + uint32_t(row & 7) * 128u + (uint32_t(chunk ^ (row & 7)) << 4);
}
constexpr uint64_t kDescriptorBase = (uint64_t(1) << 46) | (uint64_t(2) << 61) | (uint64_t(kGroupBytes >> 4) << 32);
__device__ __forceinline__ uint64_t k_major_descriptor(uint32_t smem) {
    return kDescriptorBase | (uint64_t(1) << 16) | ((smem >> 4) & 0x3fffu);
}
// column_group_bytes: distance between neighbouring groups of 64 columns.
__device__ __forceinline__ uint64_t mn_major_descriptor(uint32_t smem, uint32_t column_group_bytes) {
    return kDescriptorBase | (uint64_t((column_group_bytes >> 4) & 0x3fffu) << 16) | ((smem >> 4) & 0x3fffu);
}
// Bytes from one 16 in K to the next.
constexpr uint32_t kMajorStep = 32, mnMajorStep = 2 * kGroupBytes;
// fp16 x fp16 -> fp32, each operand along K or across it.
__host__ __device__ constexpr uint32_t f16_instruction(int m, int n, bool a_mn_major, bool b_mn_major) {
    return (1u << 4) | (a_mn_major ? 1u << 15 : 0u) | (b_mn_major ? 1u << 16 : 0u) | (uint32_t(n >> 3) << 17) | (uint32_t(m >> 4) << 24);
}

__device__ __forceinline__ void tmem_alloc(uint32_t* address_smem, uint32_t columns) {       // one warp of each CTA of the pair
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(address_smem)), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
}
__device__ __forceinline__ void tmem_free(uint32_t address, uint32_t columns) {              // the same warps
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(address), "r"(columns));
}
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t instruction, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(instruction),
        "r"(uint32_t(accumulate))
        : "memory");
}
// `bar` of both CTAs gets one arrival when every MMA this thread has issued is complete.
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)),
                 "h"(uint16_t(3))
                 : "memory");
}
// One arrival on the barrier at the same place in CTA `rank` of the cluster.
__device__ __forceinline__ void mbar_arrive_at(uint64_t* bar, uint32_t rank) {
    asm volatile(
        "{\n\t.reg .b32 a;\n\t"
        "mapa.shared::cluster.u32 a, %0, %1;\n\t"
        "mbarrier.arrive.release.cluster.shared::cluster.b64 _, [a];\n\t}" ::"r"(smem_u32(bar)),
        "r"(rank)
        : "memory");
}
// mbar_wait_bounded for a barrier on which threads of another CTA of the cluster arrive.
__device__ __forceinline__ bool mbar_wait_cluster(uint64_t* bar, unsigned parity, int max_polls = (1 << 22)) {
    const uint32_t addr = smem_u32(bar);
    for (int it = 0; it < max_polls; ++it) {
        uint32_t done;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(done)
            : "r"(addr), "r"(parity)
            : "memory");
        if (done) return true;
    }
    report_check(CHECK_MBARRIER_TIMEOUT);
    return false;
}
// The same for one CTA alone (a kernel uses either these or those above).
__device__ __forceinline__ void tmem_alloc_single(uint32_t* address_smem, uint32_t columns) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(address_smem)), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void tmem_free_single(uint32_t address, uint32_t columns) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(address), "r"(columns));
}
__device__ __forceinline__ void mma_f16_single(uint32_t d, uint64_t a, uint64_t b, uint32_t instruction, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(instruction),
        "r"(uint32_t(accumulate))
        : "memory");
}
__device__ __forceinline__ void mma_commit_single(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

__device__ __forceinline__ void tmem_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// 32 fp32 columns of the warp's 32 lanes (the thread's lane); complete after tmem_wait.
__device__ __forceinline__ void tmem_request32(uint32_t address, float (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]),
          "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]),
          "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]),
          "=f"(v[31])
        : "r"(address)
        : "memory");
}
// The values are named so that nothing reads them before the wait.
__device__ __forceinline__ void tmem_wait(float (&v)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]), "+f"(v[8]), "+f"(v[9]),
                   "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15])
                 :
                 : "memory");
    asm volatile("" : "+f"(v[16]), "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]), "+f"(v[21]), "+f"(v[22]), "+f"(v[23]), "+f"(v[24]),
                 "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]), "+f"(v[29]), "+f"(v[30]), "+f"(v[31]) : : "memory");
}
__device__ __forceinline__ void tmem_load32(uint32_t address, float (&v)[32]) {
    tmem_request32(address, v);
    tmem_wait(v);
}
__device__ __forceinline__ void tmem_load32(uint32_t address, float (&v)[32], uint32_t other_address, float (&other)[32]) {
    tmem_request32(address, v);
    tmem_request32(other_address, other);
    tmem_wait(v);
    tmem_wait(other);
}

}  // namespace gmc
